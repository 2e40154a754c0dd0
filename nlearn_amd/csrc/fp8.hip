// fp8.hip — 8-bit floating point with a scale for each block of 128: quantisation
// and the matrix product, for gfx950.
//
//   x[r, c] ~ 2^e[r / g, c / 128] * q[r, c],   q in e4m3 (OCP, largest value 448)
//   e = the least integer with max|x| over the block <= 448 * 2^e   (0 for a block of zeros)
//   C[m, n] = sum_b 2^(ea[m, b] + eb[n, b]) * sum_{k in block b} qa[m, k] qb[n, k]
//
// A power of two as scale leaves one rounding (to e4m3, to nearest even) and is
// what the matrix unit applies itself: v_mfma_scale_f32_32x32x64_f8f6f4 takes an
// e8m0 byte per row of each operand, so a block's scale costs no vector
// instruction.
//
// The 8-bit matrix instructions cut 8 products at a time to a grid of 2^-13 of
// the largest one's power of two before they add them up (measured: beside 2^16 a
// product keeps its multiples of 8; the sums of 8 are then added in fp32). On
// normal values that leaves a relative error of 1.5e-5, on values spread over the
// whole range of e4m3 7e-5: a hundredth to a twentieth of the rounding of a bf16
// result, but not the sum that an fp32 result stands for. A product with an fp32
// result therefore widens its operands to bf16 in registers (exact, with the
// scale) and takes v_mfma_f32_32x32x16_bf16, whose sums are fp32, at half the rate.
#include <type_traits>

#include "fp8.h"

namespace nl {
namespace {

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8;

// ===========================================================================
// Quantisation
// ===========================================================================

struct QuantArgs {
  int64_t rows, cols;
  const void* x;
  int64_t ldx;
  int group;    // rows per scale: 1 or 128
  uint8_t* q;   // blocks along the columns (may be null)
  int64_t ldq;
  uint8_t* s;
  int64_t lds;
  uint8_t* qt;  // the transpose, blocks along the rows (may be null)
  int64_t ldqt;
  uint8_t* st;
  int64_t ldst;
  // a layer's output gradient: x * act'(u) is quantised
  const void* u = nullptr;  // in the type of x
  int64_t ldu = 0;
  int act = NL_ACT_NONE;
  float* part = nullptr;    // column sums of each 128 rows, [ceil(rows / 128)][cols] (may be null)
};

// x between -c and c, NaN as it is (fminf and fmaxf pass it over)
__device__ __forceinline__ float clamp_nan(float x, float c) {
  return __builtin_elementwise_minimum(__builtin_elementwise_maximum(x, -c), c);
}
// The derivatives of gelu_tanh and silu from their sigmoid s (common.h), s + s (1 - s) u q with s (1 - s) =
// s - s^2 by one fma (q = 1 of silu, which beyond |u| = 120 is below 2^-166 or 1).
__device__ __forceinline__ float gelu_grad_of(float u) {
  const float s = __builtin_amdgcn_rcpf(gelu_sigmoid_arg(u));
  return __builtin_fmaf(__builtin_fmaf(-s, s, s), u * __builtin_fmaf(kGeluD2, u * u, kGeluD1), s);
}
__device__ __forceinline__ float silu_grad_of(float u) {
  const float s = __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * u));
  return __builtin_fmaf(__builtin_fmaf(-s, s, s), u, s);
}
// v *= act'(u), u of a row's `left` elements; a u that is NaN gives NaN, and relu passes or drops v whatever it is
template <typename T, int R>
__device__ __forceinline__ void scale_by_act_grad(float (&v)[R][8], const Vec<T> (&u)[R], int left, int act) {
  auto each = [&](auto scaled) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float f[8];
      unpack(u[i], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = scaled(v[i][k], f[k]);
    }
  };
  if (act == NL_ACT_GELU) each([](float g, float x) { return g * gelu_grad_of(clamp_nan(x, 20.f)); });
  else if (act == NL_ACT_SILU) each([](float g, float x) { return g * silu_grad_of(clamp_nan(x, 120.f)); });
  else each([](float g, float x) { return x > 0.f ? g : x == x ? 0.f : x; });
  if (left < 8) {  // (not by what u holds behind the row)
#pragma unroll
    for (int i = 0; i < R; ++i) clear_tail(v[i], left);
  }
}

// row[c0 .. c0+7] of a matrix of a.rows x a.cols with rows of ld, as it is stored (what is not there: see load_row)
template <typename T>
__device__ __forceinline__ Vec<T> load8(const QuantArgs& a, const void* x, int64_t ld, int64_t row, int64_t c0) {
  const int64_t left = row < a.rows ? a.cols - c0 : 0;
  return load_row(reinterpret_cast<const T*>(x) + row * ld + c0, (int)(left < 8 ? left : 8),
                  a.cols >= 8 && row + 1 < a.rows);
}
// ... as floats, zero past the last row and column
template <typename T, int R>
__device__ __forceinline__ void values8(const QuantArgs& a, const Vec<T> (&w)[R], int64_t c0, float (&v)[R][8]) {
  const int64_t left = a.cols - c0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    unpack(w[i], v[i]);
    if (a.cols & 7) clear_tail(v[i], (int)(left < 8 ? left : 8));
  }
}

// One row's block of 128 per 16 lanes, 8 elements a lane: one read, one write. Bound
// by HBM: 16384 x 2048 bf16 18 us, 8192 x 8192 32.5 us (5.7 and 6.2 TB/s), rows of 2047
// 19 (40 where rows off 16 bytes were read element by element).
template <typename T, bool kAct = false>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a, uint32_t blocks, uint32_t kb) {
  const uint32_t id = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (id >= blocks) return;  // whole groups of 16 lanes leave together
  const uint32_t row = id / kb, b = id - row * kb;
  const int l = threadIdx.x & 15;
  const int64_t c0 = (int64_t)b * kB + l * 8;
  float x[1][8];
  const Vec<T> w[1] = {load8<T>(a, a.x, a.ldx, row, c0)};
  if (kAct && a.act != NL_ACT_NONE) {
    const Vec<T> u[1] = {load8<T>(a, a.u, a.ldu, row, c0)};
    values8<T>(a, w, c0, x);
    scale_by_act_grad(x, u, (int)(a.cols - c0 < 8 ? a.cols - c0 : 8), a.act);
  } else {
    values8<T>(a, w, c0, x);
  }
  const float(&v)[8] = x[0];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
  if (m >= kInfBits) {  // look again for what is finite
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, finite_abs_bits(v[i]));
  }
  const int byte = scale_byte(max16(m));
  *reinterpret_cast<u32x2*>(a.q + (int64_t)row * a.ldq + c0) =
      u32x2{pack_e4m3x4(v[0], v[1], v[2], v[3], byte), pack_e4m3x4(v[4], v[5], v[6], v[7], byte)};
  if (l == 0) a.s[(int64_t)row * a.lds + b] = (uint8_t)byte;
}

// max over the lanes l, l + 16, l + 32, l + 48
__device__ __forceinline__ uint32_t max_rows(uint32_t v) {
  const auto r16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max((uint32_t)r16[0], (uint32_t)r16[1]);
  const auto r32 = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)r32[0], (uint32_t)r32[1]);
}

// sum over the lanes l, l + 16, l + 32, l + 48
__device__ __forceinline__ float sum_rows(float v) {
  const uint32_t a = __float_as_uint(v);
  const auto r16 = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  v = __uint_as_float(r16[0]) + __uint_as_float(r16[1]);
  const uint32_t b = __float_as_uint(v);
  const auto r32 = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __uint_as_float(r32[0]) + __uint_as_float(r32[1]);
}

// A 128 x 128 tile per workgroup: read once, written along the rows and, through
// LDS, along the columns. Lane group g = tid / 16 holds rows 4g .. 4g+3, lane
// l = tid % 16 columns 8l .. 8l+7, so a thread has 4 bytes of a column that lie
// together in the transpose. Column c's dword g is at slot g ^ 4 (c / 8 % 8): 16-byte
// pieces stay whole, and 8 lanes' columns fall on different banks.
// Bound by HBM: 16384 x 2048 bf16 26.5 us (5.1 TB/s), 16384 x 2047 29, an fp32 weight of
// 512 x 50257 in padded rows 31.7 us, in dense ones 35 (31, 53 and 62 where each row's loads
// were waited for before the next row's, those off 16 bytes element by element); with 256
// threads of twice the elements, each looked at twice for values that are not finite, whole
// and padded rows took 33.1 and 31.9 us. A layer's x and W go in one launch: 777 x 1000 x 333
// forward 22.3 us, in two 26.7; 16384 x 2048 x 512 48.2 and 52.5.
struct QuantTile {
  uint32_t tile[kB * 32];
  uint32_t colmax[8][kB];
  uint8_t colbyte[kB];
};
template <typename T, bool kAct = false>
__device__ __forceinline__ void quantize_tile(const QuantArgs& a, uint32_t block, uint32_t cb, QuantTile& sm) {
  auto& tile = sm.tile;
  auto& colmax = sm.colmax;
  auto& colbyte = sm.colbyte;
  const int tid = threadIdx.x, l = tid & 15, g = tid >> 4;
  const uint32_t by = block / cb, bx = block - by * cb;
  const int64_t r0 = (int64_t)by * kB, c0 = (int64_t)bx * kB;
  const int64_t cl = c0 + l * 8;
  float v[4][8];
  const bool with_u = kAct && a.act != NL_ACT_NONE;
  Vec<T> w[4], u[kAct ? 4 : 1];
  if (r0 + kB <= a.rows && c0 + kB <= a.cols) {  // a whole tile
    // every load is out before the first one is waited for
    auto load4 = [&](const void* x, int64_t ld, Vec<T> (&o)[4]) __attribute__((always_inline)) {
      const T* p = reinterpret_cast<const T*>(x) + (r0 + g * 4) * ld + cl;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = load_vec(p + i * ld, 8);
    };
    load4(a.x, a.ldx, w);
    if constexpr (kAct)
      if (with_u) load4(a.u, a.ldu, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack(w[i], v[i]);
    if constexpr (kAct)
      if (with_u) scale_by_act_grad(v, u, 8, a.act);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = load8<T>(a, a.x, a.ldx, r0 + g * 4 + i, cl);
    if constexpr (kAct)
      if (with_u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = load8<T>(a, a.u, a.ldu, r0 + g * 4 + i, cl);
      }
    values8<T>(a, w, cl, v);
    if constexpr (kAct)
      if (with_u) scale_by_act_grad(v, u, (int)(a.cols - cl < 8 ? a.cols - cl : 8), a.act);
  }
  if constexpr (kAct) {
    if (a.part) {  // the tile's column sums: a thread's 4 rows, a wave's 4 groups, then the 8 waves
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = sum_rows((v[0][j] + v[1][j]) + (v[2][j] + v[3][j]));
        if ((tid & 63) < 16) colmax[tid >> 6][l * 8 + j] = __float_as_uint(t);
      }
      __syncthreads();
      if (tid < kB && c0 + tid < a.cols) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += __uint_as_float(colmax[i][tid]);
        a.part[(int64_t)by * a.cols + c0 + tid] = t;
      }
      __syncthreads();
    }
  }
  uint32_t rm[4], cm[8];
  auto maxima = [&](auto bits) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) cm[j] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      rm[i] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t u = bits(v[i][j]);
        rm[i] = max(rm[i], u);
        cm[j] = max(cm[j], u);
      }
    }
  };
  maxima([](float x) { return abs_bits(x); });
  if (max(max(rm[0], rm[1]), max(rm[2], rm[3])) >= kInfBits)  // look again for what is finite
    maxima([](float x) { return finite_abs_bits(x); });
  if (a.group != 1 || a.qt) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t m = max_rows(cm[j]);
      if ((tid & 63) < 16) colmax[tid >> 6][l * 8 + j] = m;
    }
    __syncthreads();
    if (tid < kB) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, colmax[i][tid]);
      if (a.group == 1) colbyte[tid] = (uint8_t)scale_byte(m);
      else colmax[0][tid] = m;  // this thread alone read column tid
    }
    __syncthreads();
  }
  int one = 0;
  if (a.group != 1) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, colmax[0][l * 8 + j]);
    one = scale_byte(max16(m));
  }
  if (a.q) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = r0 + g * 4 + i;
      const int byte = a.group != 1 ? one : scale_byte(max16(rm[i]));
      if (r >= a.rows) continue;
      const float* w = v[i];
      *reinterpret_cast<u32x2*>(a.q + r * a.ldq + cl) =
          u32x2{pack_e4m3x4(w[0], w[1], w[2], w[3], byte), pack_e4m3x4(w[4], w[5], w[6], w[7], byte)};
      if (l == 0 && a.group == 1) a.s[r * a.lds + bx] = (uint8_t)byte;
    }
    if (a.group != 1 && tid == 0) a.s[(int64_t)by * a.lds + bx] = (uint8_t)one;
  }
  if (!a.qt) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = l * 8 + j;
    tile[c * 32 + (g ^ ((l & 7) << 2))] =
        pack_e4m3x4(v[0][j], v[1][j], v[2][j], v[3][j], a.group != 1 ? one : colbyte[c]);
  }
  __syncthreads();
  // 8 lanes write a column's 128 bytes, 16 a lane
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int c = it * 64 + (tid >> 3), h = tid & 7;
    if (c0 + c >= a.cols) continue;
    *reinterpret_cast<u32x4*>(a.qt + (c0 + c) * a.ldqt + r0 + h * 16) =
        *reinterpret_cast<const u32x4*>(tile + c * 32 + ((h ^ ((c >> 3) & 7)) << 2));
  }
  if (a.group == 1) {
    if (tid < kB && c0 + tid < a.cols) a.st[(c0 + tid) * a.ldst + by] = colbyte[tid];
  } else if (tid == 0) {
    a.st[(int64_t)bx * a.ldst + by] = (uint8_t)one;
  }
}

// With an activation 16384 x 2048 bf16 takes 43 us (gelu; relu 42, none 26.5), 46 with the column sums
// and their own launch: 201 MB at 4.7 TB/s, near the rate of the tile without one. Row by row, each row's load
// waited for before the next one's, it was 47 and 31. 128 registers are two workgroups a CU; with 138,
// one, it took 71, and held to 80, three, it spilled (91; without an activation 31 for 28). Stores past
// the caches gained 3 alone and lost 10 us in the layer, whose products read them next.
template <typename T, bool kAct = false>
__global__ __launch_bounds__(512, kAct ? 4 : 2) void quantize_tile_kernel(QuantArgs a, uint32_t cb) {
  __shared__ __attribute__((aligned(16))) QuantTile sm;
  quantize_tile<T, kAct>(a, blockIdx.x, cb, sm);
}

// Two matrices in one launch, the first one's tiles (na of them) before the second's.
template <typename TA, typename TB>
__global__ __launch_bounds__(512) void quantize_two_kernel(QuantArgs a, uint32_t cba, uint32_t na, QuantArgs b,
                                                           uint32_t cbb) {
  __shared__ __attribute__((aligned(16))) QuantTile sm;
  if (blockIdx.x < na) quantize_tile<TA>(a, blockIdx.x, cba, sm);
  else quantize_tile<TB>(b, blockIdx.x - na, cbb, sm);
}

// ===========================================================================
// Product
// ===========================================================================
//
// Both operands have the summed axis contiguous, in whole blocks of 128 (the last
// one padded with zeros), so a K step of 128 is one block and one scale per row.
//   * Tiles go global -> LDS by DMA, [row][128 bytes] with the 16-byte chunks of
//     a row XOR-swizzled, in two stages with one barrier each.
//   * A lane's fragment of 32 x 64 is 32 bytes of row lane % 32: two ds_read_b128.
//     Which k a byte stands for does not matter as long as both operands agree
//     and the scale holds for all 128.
//   * The lane's scale bytes of four K steps come as one dword per 32 rows.
//   * Operands are swapped (B as src A), so a lane ends up with 4 consecutive
//     columns; rows leave through LDS in whole 16-byte pieces (stored from the lanes
//     as they are, in pieces of 32 bytes a row, 16384 x 50257 x 512 took 672 us for 515).
//   * 256 x 256 tiles run 4 waves of 128 x 128, one a SIMD: 256 accumulator registers
//     and two sets of fragments (128) in the 512 it has, and two thirds of the LDS
//     reads of 8 waves of 128 x 64, which with the DMA's writes would take as long as
//     the MFMAs.
// Measured: 8192^3 to bf16 374 us over the same operands again and 409 over new ones each
// time, 2.94 and 2.69 PFLOP/s (a library's product with one scale a tensor 3.03): the MFMAs
// are busy 72 to 77% of the cycles, at the 1.55 to 1.62 GHz that the part holds under them;
// the rest is the meeting of the waves at each stage and the tiles' stores. To fp32 (widened)
// 725 us, 1.52 PFLOP/s. Scale rows that are no whole dwords cost 2% (4096 x 4096 x 4992: 68.9
// us for 67.3; to fp32 122.6 for 122.4). 16384 x 50257 x 512, four stages a
// tile: 466 to 491 us by card, some 100 fewer without its stores: 1.65 GB go out in bursts
// between K loops that the next tile's first two stages hide in part. The stores pass
// the caches by (not so, 16384 x 50257 x 512 took 569 us for 489, and the products of a
// 16384 x 512 x 2048 layer with its gradients 137 us for 132).

struct GemmF8Args {
  int M, N, K, Kp;
  const uint8_t* A;
  int64_t lda;
  const uint8_t* sa;
  int64_t ldsa;
  int sha;  // log2 of the rows per scale: 0 or 7
  const uint8_t* B;
  int64_t ldb;
  const uint8_t* sb;
  int64_t ldsb;
  int shb;
  int dw;  // scale rows of both are whole, aligned dwords
  void* C;
  int64_t ldc;
  float* ws;     // split partials [splits][M][ldw], or null
  int64_t ldw;
  int tiles;     // output tiles
  int items;     // tiles * splits
  int kb_chunk;  // blocks per split (a multiple of 4 when there is more than one)
  // the epilogue's, of the kernels that have one
  const void* bias;   // fp32 or (bias16) bf16, may be null
  int bias16;
  int act;            // NL_ACT_*
  const void* res;    // in the type of C (bf16 beside 8 bits), may be null
  int64_t ldres;
  void* aux;          // u in the type of C, may be null
  int64_t ldaux;
  uint8_t* sc;        // scales of C in 8 bits
  int64_t ldsc;
};

// Epilogues of a product: none; u = acc + bias, C = act(u); that with u rounded to the type of C
// before, and kept where it is asked for (what a backward pass reads); each with a residual.
// All of it is done in the lanes as the matrix unit leaves the sums, and only what is stored passes
// the slab: bias and activation on rows read back from an fp32 slab took 39 us to bf16 and 51 to 8
// bits for 16384 x 2048 x 512 with gelu. Measured (us; without an epilogue 27): bias to bf16 27, with
// gelu 34, with u kept 39 (two results of 67 MB), a residual 36; to 8 bits 27, with gelu 33; to fp32
// with gelu 50 (without an epilogue 46). 8192^3: 403 without, silu or gelu to bf16 410, to 8 bits
// 424, a residual 430 to 444. With K = 512 a tile's sums take as long as its epilogue (gelu: 12
// vector instructions an element to 8 bits, about 14 us of the chip's issue beside 13 us of the
// matrix units), and two workgroups a CU hide half of that; starting them half a tile apart changed nothing.
// On 256 x 256 tiles a group's values, the residual's pieces and the next item's first fragments live beside the
// sums, and registers go to scratch: with a residual 52 to 54 of a result in 8 bits, 3 to 11 of bf16 and up to 1 of
// fp32; fp32 with u kept 28 to 34, 8 bits without a residual 6. The other forms and all of 128 x 128 keep theirs.
enum { kPlain = 0, kEpi = 1, kEpiKeep = 2, kEpiRes = 3, kEpiResKeep = 4 };
constexpr bool keeps(int epi) { return epi == kEpiKeep || epi == kEpiResKeep; }

// Four scale bytes of one row from byte `off` (n of them there): one dword where
// rows are whole, aligned dwords, else byte by byte.
template <bool kDw>
__device__ __forceinline__ uint32_t scales4(__amdgpu_buffer_rsrc_t rs, uint32_t off, int n) {
  if constexpr (kDw) {
    return __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
  } else {
    uint32_t v = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      v |= (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(rs, b < n ? off + b : 0xffffffffu, 0, 0) << (8 * b);
    return v;
  }
}

// 16 e4m3 bytes times a power of two (given as its scale byte in a float's exponent) to two
// fragments of 8 bf16: 4 significant bits in 8. Exact for scale bytes 3 to 246, with which
// 2^-9 is at bf16's least subnormal, 2^-133, and 448 below its largest value. Below, values of
// e4m3's subnormals lose bits; above, values of 2^128 and more are infinite. No share of the
// exponent can be moved to the result: a lane's rows have scales of their own in every block.
__device__ __forceinline__ void widen(const u32x4& v, float scale, bf16x8 out[2]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)v[i], scale, false));
    w[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)v[i], scale, true));
  }
  out[0] = as_bf16x8(u32x4{w[0], w[1], w[2], w[3]});
  out[1] = as_bf16x8(u32x4{w[4], w[5], w[6], w[7]});
}

// Slot of 16-byte chunk c of row r: c ^ swz(r). 16 consecutive rows at one chunk (a
// fragment read) fall on all 64 banks, and rows 16 apart share the swizzle.
__device__ __forceinline__ int swz(int r) { return (r & 7) ^ ((r >> 3) & 1); }

// A lane's fragment: 16 bytes to widen, or the 32 that an 8-bit MFMA takes.
template <bool kWide>
struct FragOf {
  typedef u32x4 type;
};
template <>
struct FragOf<false> {
  typedef i32x8 type;
};
template <bool kWide>
__device__ __forceinline__ typename FragOf<kWide>::type read_frag(const uint8_t* p, const int* off) {
  const u32x4 lo = *reinterpret_cast<const u32x4*>(p + off[0]);
  if constexpr (kWide) {
    return lo;
  } else {
    const u32x4 hi = *reinterpret_cast<const u32x4*>(p + off[1]);
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  }
}

// One MFMA, then its share of the R fragment reads of the next step and of the D
// DMA instructions of a stage.
template <int M, int NM, int R, int D>
__device__ __forceinline__ void sched_f8() {
  if constexpr (M < NM) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    constexpr int lo = M * R / NM, hi = (M + 1) * R / NM;
    if constexpr (hi > lo) __builtin_amdgcn_sched_group_barrier(0x100, hi - lo, 0);
    constexpr int dlo = M * D / NM, dhi = (M + 1) * D / NM;
    if constexpr (dhi > dlo) __builtin_amdgcn_sched_group_barrier(0x010, dhi - dlo, 0);
    sched_f8<M + 1, NM, R, D>();
  }
}

// A workgroup (one per CU with 256 x 256 tiles, two with 128 x 128) walks its items
// (a tile's share of K) without a pause in the operand stream: an item's last two
// stages start the DMA of the next item's first two, and its stores drain while the
// next item's first stages compute.
struct F8Item {
  int m0, n0, split, kb0, nkb;  // nkb: blocks of K
  const uint8_t *a, *b, *sa, *sb;
  uint32_t ba, bb, bsa, bsb;    // bytes in reach of each (0: no such item)
};

// the bytes that a descriptor of a tile reaches, and an offset past them, for stores that
// are dropped: 16 bytes from there do not pass 2^32 either
constexpr uint32_t kNowhere = 0xfffffff0u;

// the same on every lane, and known to be
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = (uint64_t)p;
  return reinterpret_cast<const uint8_t*>((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

template <int BM, int BN>
__device__ __forceinline__ F8Item f8_item(const GemmF8Args& g, int item) {
  F8Item t;
  const int tiles_n = (g.N + BN - 1) / BN;
  const int tiles_m = (g.M + BM - 1) / BM;
  item = uniform(item);
  t.split = item / g.tiles;
  const int tile = item - t.split * g.tiles;
  // tile rows that neighbours share a column of B over (16384 x 50257 x 512 and 8192^3, us on
  // one card: 1 row 516 and 411, 4 464 and 367, 8 464 and 372, 16 464 and 382)
  constexpr int GM = 8;
  const int in_group = GM * tiles_n;
  const int first_m = (tile / in_group) * GM;
  const int gsize = min(tiles_m - first_m, GM);
  t.m0 = (first_m + (tile % in_group) % gsize) * BM;
  t.n0 = ((tile % in_group) / gsize) * BN;
  t.kb0 = t.split * g.kb_chunk;
  t.nkb = min(g.Kp / kB, t.kb0 + g.kb_chunk) - t.kb0;
  // Descriptors start at the item's first row (64-bit base), so 32-bit offsets reach
  // any matrix; rows past the last one read as zero.
  const int ra = min(g.M - t.m0, BM), rb = min(g.N - t.n0, BN);
  t.a = g.A + (int64_t)t.m0 * g.lda;
  t.b = g.B + (int64_t)t.n0 * g.ldb;
  t.sa = g.sa + (int64_t)(t.m0 >> g.sha) * g.ldsa + t.kb0;
  t.sb = g.sb + (int64_t)(t.n0 >> g.shb) * g.ldsb + t.kb0;
  t.ba = (uint32_t)((int64_t)(ra - 1) * g.lda + g.Kp);
  t.bb = (uint32_t)((int64_t)(rb - 1) * g.ldb + g.Kp);
  // whole dwords of scales where rows hold them (the last one may end in padding); none
  // without a block (K == 0, where the operands' pointers may be null)
  t.bsa = t.nkb == 0 ? 0 : (uint32_t)(((ra - 1) >> g.sha) * g.ldsa + (g.dw ? (t.nkb + 3) / 4 * 4 : t.nkb));
  t.bsb = t.nkb == 0 ? 0 : (uint32_t)(((rb - 1) >> g.shb) * g.ldsb + (g.dw ? (t.nkb + 3) / 4 * 4 : t.nkb));
  return t;
}

// act(u) of some values; NaN stays NaN
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  if (act == NL_ACT_GELU) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = gelu_tanh(v[k]);
  } else if (act == NL_ACT_SILU) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = silu(v[k]);
  } else if (act == NL_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = v[k] < 0.f ? 0.f : v[k];
  }
}

// kDw: scale rows are whole, aligned dwords. Else a scale dword is four byte loads.
// OutT: float, uint16_t (bf16) or, with an epilogue, uint8_t (e4m3 with its scales). kWide: widened
// to bf16 for fp32 sums.
template <int BM, int BN, int WTM, int WTN, typename OutT, bool kDw, int EPI = kPlain, bool kWide = sizeof(OutT) == 4>
__global__ __launch_bounds__((BM / WTM) * (BN / WTN) * 64, (BM * BN >= 65536) ? 1 : 2) void gemm_f8_kernel(
    GemmF8Args g) {
  constexpr int WNW = BN / WTN, NWV = (BM / WTM) * WNW;
  constexpr int FM = WTM / 32, FN = WTN / 32;
  constexpr int STAGE = (BM + BN) * kB;
  constexpr int IA = BM / 8 / NWV, IB = BN / 8 / NWV;  // DMA instructions (8 rows each) per wave and stage
  static_assert(IA * 8 * NWV == BM && IB * 8 * NWV == BN, "a stage splits into whole DMA instructions");
  constexpr int NS = kWide ? 4 : 2;                    // fragment steps of a stage: 16 or 32 bytes of k a lane
  constexpr int CH = kWide ? 1 : 2;                    // 16-byte chunks of a fragment
  // bytes of a slab row: WTN bf16 or half as many fp32
  constexpr int PITCH = BM * BN >= 65536 || 2 * WTN < 128 ? 2 * WTN : 128;
  static_assert(PITCH == 2 * WTN || EPI != kPlain, "an item without an epilogue leaves in slabs of whole rows");
  // Each stage is an LDS object of its own: the compiler then knows that the DMA into
  // one does not alias the reads of the other.
  __shared__ __attribute__((aligned(16))) uint8_t st0[STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t st1[STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t slabs[NWV * 32 * PITCH];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WNW, wn = wave % WNW;

  // Items of this workgroup: each XCD takes a contiguous run of them (neighbours share
  // rows of A and B in its L2), its workgroups take turns within it.
  const int nx = gridDim.x >= 8 ? 8 : 1;
  const int xcd = blockIdx.x % nx, turn = blockIdx.x / nx;
  const int wgs = (gridDim.x - xcd + nx - 1) / nx;
  const int share = g.items / nx, odd = g.items % nx;  // the first `odd` XCDs have one item more, as they have workgroups
  int item = xcd * share + min(xcd, odd);
  const int last = item + share + (xcd < odd ? 1 : 0);
  item += turn;
  if (item >= last) return;

  uint32_t va[IA], vb[IB];
#pragma unroll
  for (int i = 0; i < IA; ++i) {
    const int r = (i * NWV + wave) * 8 + (lane >> 3);
    va[i] = (uint32_t)((int64_t)r * g.lda) + (((lane & 7) ^ swz(r)) << 4);
  }
#pragma unroll
  for (int i = 0; i < IB; ++i) {
    const int r = (i * NWV + wave) * 8 + (lane >> 3);
    vb[i] = (uint32_t)((int64_t)r * g.ldb) + (((lane & 7) ^ swz(r)) << 4);
  }
  // the DMA of an item's stage kt; behind its last block an empty descriptor gives zeros
  auto issue = [&](uint8_t* sb, const F8Item& t, int kt) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(uniform(t.a), uniform(kt < t.nkb ? t.ba : 0));
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(uniform(t.b), uniform(kt < t.nkb ? t.bb : 0));
    const uint32_t soff = uniform((t.kb0 + kt) * kB);
#pragma unroll
    for (int i = 0; i < IA; ++i) dma16(ra, sb + (i * NWV + wave) * 1024, va[i], soff);
#pragma unroll
    for (int i = 0; i < IB; ++i) dma16(rb, sb + BM * kB + (i * NWV + wave) * 1024, vb[i], soff);
  };

  // Scale bytes of this lane's rows, four blocks to a dword; rows and blocks that are
  // not there read as 0 (2^-127, against values of zero).
  const int frow = lane & 31;
  uint32_t osa[FM], osb[FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) osa[i] = (uint32_t)(((wm * WTM + i * 32 + frow) >> g.sha) * g.ldsa);
#pragma unroll
  for (int j = 0; j < FN; ++j) osb[j] = (uint32_t)(((wn * WTN + j * 32 + frow) >> g.shb) * g.ldsb);
  uint32_t sca[FM], scb[FN], nca[FM], ncb[FN];
  auto load_scales = [&](const F8Item& t, int q) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(uniform(t.sa), uniform(t.bsa));
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(uniform(t.sb), uniform(t.bsb));
#pragma unroll
    for (int i = 0; i < FM; ++i) nca[i] = scales4<kDw>(ra, osa[i] + 4 * q, t.nkb - 4 * q);
#pragma unroll
    for (int j = 0; j < FN; ++j) ncb[j] = scales4<kDw>(rb, osb[j] + 4 * q, t.nkb - 4 * q);
  };
  // n: the blocks that the set holds. What stands behind them in the last dword is not
  // a scale, and could be a NaN.
  auto take_scales = [&](int n) __attribute__((always_inline)) {
    const uint32_t there = n >= 4 ? ~0u : (1u << (8 * n)) - 1u;
#pragma unroll
    for (int i = 0; i < FM; ++i) sca[i] = nca[i] & there;
#pragma unroll
    for (int j = 0; j < FN; ++j) scb[j] = ncb[j] & there;
  };

  // fragment (i, step t): row i * 32 + frow, chunks of step t; one offset per step and chunk
  int offa[NS][CH], offb[NS][CH];
#pragma unroll
  for (int t = 0; t < NS; ++t)
#pragma unroll
    for (int h = 0; h < CH; ++h) {
      const int c = (t * 2 + (lane >> 5)) * CH + h;
      const int o = frow * kB + ((c ^ swz(frow)) << 4);
      offa[t][h] = wm * WTM * kB + o;
      offb[t][h] = (BM + wn * WTN) * kB + o;
    }
  using Frag = typename FragOf<kWide>::type;
  Frag fa[2][FM], fb[2][FN];
  auto read = [&](const uint8_t* sb, int t, int into) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[into][j] = read_frag<kWide>(sb + j * 32 * kB, offb[t]);
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[into][i] = read_frag<kWide>(sb + i * 32 * kB, offa[t]);
  };

  f32x16 acc[FM][FN];
  auto compute = [&](int in, auto pos, auto first) __attribute__((always_inline)) {
    constexpr int P = decltype(pos)::value;  // the block's byte in the scale dwords
    constexpr bool kFirst = decltype(first)::value;
    f32x16 zero;
#pragma unroll
    for (int r = 0; r < 16; ++r) zero[r] = 0.f;
    if constexpr (kWide) {
      bf16x8 b[FN][2];
#pragma unroll
      for (int j = 0; j < FN; ++j) widen(fb[in][j], __uint_as_float((scb[j] >> (8 * P) & 0xff) << 23), b[j]);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        bf16x8 a[2];
        widen(fa[in][i], __uint_as_float((sca[i] >> (8 * P) & 0xff) << 23), a);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma32(b[j][h], a[h], kFirst && h == 0 ? zero : acc[i][j]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
              fb[in][j], fa[in][i], kFirst ? zero : acc[i][j], 0, 0, P, (int)scb[j], P, (int)sca[i]);
    }
  };

  // Stage kt: every step reads the next one's fragments while its MFMAs run. The
  // last step's fragments are in registers when the workgroup meets, so the stage's
  // buffer is free for the stage after next (its own item's or the next one's), and
  // the first fragments of the next stage, whose DMA has had a whole stage to land,
  // are read under the last step's MFMAs. (No branch stands between MFMAs: the
  // compiler would move those before it to the ones behind it.)
  F8Item cur = f8_item<BM, BN>(g, item), nxt = cur;
  int stages = 0;  // of the current item: an even number, the last one of zeros with an odd one of blocks
  auto stage = [&](int kt, auto pos, auto first, auto wait) __attribute__((always_inline)) {
    uint8_t* here = decltype(pos)::value % 2 == 0 ? st0 : st1;
    uint8_t* there = decltype(pos)::value % 2 == 0 ? st1 : st0;
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      if (t + 1 < NS) {
        read(here, t + 1, (t + 1) & 1);
      } else {
        wait_vm<decltype(wait)::value>();
        __syncthreads();
        const bool own = kt + 2 < stages;
        F8Item ahead = cur;
        ahead.a = own ? cur.a : nxt.a;
        ahead.b = own ? cur.b : nxt.b;
        ahead.ba = own ? cur.ba : nxt.ba;
        ahead.bb = own ? cur.bb : nxt.bb;
        ahead.kb0 = own ? cur.kb0 : nxt.kb0;
        ahead.nkb = own ? cur.nkb : nxt.nkb;
        issue(here, ahead, own ? kt + 2 : kt + 2 - stages);
        read(there, 0, 0);
      }
      if (t == 0) compute(0, pos, first);
      else compute(t & 1, pos, std::false_type{});
      if constexpr (kWide) {
        if (t + 1 == NS) sched_f8<0, 2 * FM * FN, 0, IA + IB>();
      } else {
        if (t + 1 < NS) sched_f8<0, FM * FN, (FM + FN) * CH, 0>();
        else sched_f8<0, FM * FN, (FM + FN) * CH, IA + IB>();
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using P0 = std::integral_constant<int, 0>;
  using P1 = std::integral_constant<int, 1>;
  using P2 = std::integral_constant<int, 2>;
  using P3 = std::integral_constant<int, 3>;
  using No = std::false_type;
  // the scales of the four blocks behind kt's, or the next item's first
  auto scales_ahead = [&](int kt) __attribute__((always_inline)) {
    const bool own = kt + 4 < cur.nkb;
    F8Item t = cur;
    t.sa = own ? cur.sa : nxt.sa;
    t.sb = own ? cur.sb : nxt.sb;
    t.bsa = own ? cur.bsa : nxt.bsa;
    t.bsb = own ? cur.bsb : nxt.bsb;
    t.nkb = own ? cur.nkb : nxt.nkb;
    load_scales(t, own ? (kt >> 2) + 1 : 0);
  };
  constexpr int kScales = (FM + FN) * (kDw ? 1 : 4);       // loads of one set of scales
  // stores of a whole tile, 64 lanes of 16 bytes each
  constexpr int kStores = FM * 32 * WTN * (int)sizeof(OutT) / 1024;

  // bias of this wave's columns, one of each 64 a lane (0 past the last column, or without a bias)
  constexpr int kBias = EPI != kPlain ? WTN / 64 : 1;
  float bias1[kBias];
  auto load_bias = [&](const F8Item& t) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(g.bias ? g.bias : g.C, kNowhere);
    const int n = g.bias ? g.N : 0;
#pragma unroll
    for (int k = 0; k < kBias; ++k) {
      const int c = t.n0 + wn * WTN + k * 64 + lane;
      if (g.bias16)
        bias1[k] = bf16_to_f32(__builtin_amdgcn_raw_buffer_load_b16(rb, c < n ? (uint32_t)c * 2u : kNowhere, 0, 0));
      else
        bias1[k] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rb, c < n ? (uint32_t)c * 4u : kNowhere, 0, 0));
    }
  };

  load_scales(cur, 0);
  issue(st0, cur, 0);
  issue(st1, cur, 1);
  wait_vm<0>();  // both: the first stage's wait counts on the stores of an item before it
  __syncthreads();
  take_scales(cur.nkb);
  read(st0, 0, 0);
  for (;;) {
    const int next = item + wgs;
    if (next < last) {
      nxt = f8_item<BM, BN>(g, next);
    } else {
      nxt.nkb = 0;
      nxt.bsa = nxt.bsb = 0;
    }
    stages = (cur.nkb + 1) & ~1;
    // Behind this stage's DMA lie the last item's stores and this set of scales (a tile
    // at an edge has waited for its stores itself).
    scales_ahead(0);
    if constexpr (EPI != kPlain) load_bias(cur);
    stage(0, P0{}, std::true_type{}, std::integral_constant<int, (kScales + kStores < 63 ? kScales + kStores : 63)>{});
    stage(1, P1{}, No{}, P0{});
    if (stages > 2) {
      stage(2, P2{}, No{}, P0{});
      stage(3, P3{}, No{}, P0{});
      int kt = 4;
      for (; kt + 4 <= stages; kt += 4) {
        take_scales(cur.nkb - kt);
        scales_ahead(kt);
        stage(kt, P0{}, No{}, P0{});
        stage(kt + 1, P1{}, No{}, P0{});
        stage(kt + 2, P2{}, No{}, P0{});
        stage(kt + 3, P3{}, No{}, P0{});
      }
      if (kt < stages) {
        take_scales(cur.nkb - kt);
        scales_ahead(kt);
        stage(kt, P0{}, No{}, P0{});
        stage(kt + 1, P1{}, No{}, P0{});
      }
    }
    take_scales(nxt.nkb);  // landed by the last stage's wait: nothing of the next item waits for the stores below

    // Each wave passes 32 rows of PITCH bytes at a time through its own LDS slab and
    // stores rows in 16-byte pieces (a lane's own results are pieces of 32 rows).
    uint8_t* wl = slabs + wave * 32 * PITCH;
    // (hidden from the compiler, which would keep every address of the stores across
    // the loop over items, in registers that the fragments need)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int fr = ln & 31, g4 = (ln >> 5) * 4;
    // 32 rows of 64 bf16 columns of a matrix over C, at `row` and `col` of the tile, as whole 16-byte
    // pieces: 8 lanes a row. Rows and columns that are not there are out of every range (a piece that
    // N cuts is whole: rows hold N rounded up to 8).
    const int rr = ln / 8, gg = ln % 8;
    auto piece_off = [&](uint32_t ld, int rows, int cols, int row, int col) __attribute__((always_inline)) {
      return rr < rows - row && gg * 8 < cols - col ? (((uint32_t)rr + row) * ld + gg * 8 + col) * 2 : kNowhere;
    };
    auto load_rows = [&](__amdgpu_buffer_rsrc_t rs, uint32_t ld, int rows, int cols, int row, int col, u32x4 (&r)[4])
        __attribute__((always_inline)) {
#pragma unroll
      for (int it = 0; it < 4; ++it)
        r[it] = __builtin_amdgcn_raw_buffer_load_b128(rs, piece_off(ld, rows, cols, row + it * 8, col), 0, 0);
    };
    // ... added to the lanes' own values of them, through the slab
    auto add_rows = [&](const u32x4 (&r)[4], float (&v0)[16], float (&v1)[16]) __attribute__((always_inline)) {
#pragma unroll
      for (int it = 0; it < 4; ++it)
        *reinterpret_cast<u32x4*>(wl + (it * 8 + rr) * 128 + ((gg ^ rr) << 4)) = r[it];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(wl + fr * 128 + (((j * 4 + q) ^ (fr & 7)) << 4) + g4 * 2);
          float* v = (j ? v1 : v0) + 4 * q;
          v[0] += bf16_lo(w[0]), v[1] += bf16_hi(w[0]), v[2] += bf16_lo(w[1]), v[3] += bf16_hi(w[1]);
        }
    };
    if constexpr (sizeof(OutT) == 1) {
      // C in 8 bits. A wave's columns are one block of 128, and a lane pair (l, l + 32) has a whole row
      // of it: bias, activation, residual and the row's largest value in the lanes as they are, and
      // the bytes through the slab into whole rows.
      static_assert(WTN == kB && (PITCH == 256 || FM == 1), "a wave holds whole blocks of C");
      uint8_t* wb = wl + (PITCH == 256 ? 4096 : 0);  // the bias, behind the bytes or (one group of rows) before them
#pragma unroll
      for (int k = 0; k < kBias; ++k) reinterpret_cast<float*>(wb)[k * 64 + ln] = bias1[k];
      const int n = cur.n0 + wn * WTN, cols = g.N - n, rows = g.M - cur.m0;
      const bool there = cols > 0;
      const __amdgpu_buffer_rsrc_t rc = make_rsrc(
          uniform(reinterpret_cast<const uint8_t*>(g.C) + (there ? (int64_t)cur.m0 * g.ldc + n : 0)), kNowhere);
      const __amdgpu_buffer_rsrc_t rres = make_rsrc(
          uniform(reinterpret_cast<const uint8_t*>(g.res ? g.res : g.C) +
                  (g.res && there ? ((int64_t)cur.m0 * g.ldres + n) * 2 : 0)), kNowhere);
      constexpr bool kHasRes = EPI == kEpiRes;
      u32x4 res[4];
      auto load_res = [&](int i, int h) __attribute__((always_inline)) {
        load_rows(rres, (uint32_t)g.ldres, there ? rows : 0, cols, wm * WTM + i * 32, h * 64, res);
      };
      if constexpr (kHasRes) load_res(0, 0);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int row = wm * WTM + i * 32 + fr;
        float v[FN][16];
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          asm volatile("" : "+v"(acc[i][j]));  // out of the accumulators here and not before
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 b = *reinterpret_cast<const f32x4*>(wb + (j * 32 + q * 8 + g4) * 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j][4 * q + k] = acc[i][j][4 * q + k] + b[k];
          }
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) activate(v[j], g.act);
        if constexpr (kHasRes) {
          add_rows(res, v[0], v[1]);
          load_res(i, 1);
          add_rows(res, v[2], v[3]);
          if (i + 1 < FM) load_res(i + 1, 0);
        }
        if (cols < kB) {  // nothing past N has a part in the scale, and its bytes are zero
#pragma unroll
          for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (j * 32 + k / 4 * 8 + g4 + k % 4 >= cols) v[j][k] = 0.f;
        }
        // (the hardware's maximum passes a NaN over)
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int k = 0; k < 16; ++k) top = fmaxf(top, fabsf(v[j][k]));
        uint32_t m = __float_as_uint(top);
        if (__builtin_expect(__any(m >= kInfBits), 0)) {  // look again for what is finite
          m = 0;
#pragma unroll
          for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) m = max(m, finite_abs_bits(v[j][k]));
        }
        const auto r32 = __builtin_amdgcn_permlane32_swap(m, m, false, false);
        m = max((uint32_t)r32[0], (uint32_t)r32[1]);
        const int byte = scale_byte(m);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint32_t*>(wl + fr * 128 + (((2 * j + (q >> 1)) ^ (fr & 7)) << 4) + (q & 1) * 8 + g4) =
                pack_e4m3x4(v[j][4 * q], v[j][4 * q + 1], v[j][4 * q + 2], v[j][4 * q + 3], byte);
        if (ln < 32 && row < rows && there) g.sc[(int64_t)(cur.m0 + row) * g.ldsc + n / kB] = (uint8_t)byte;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int r = it * 8 + ln / 8, at = wm * WTM + i * 32 + r;
          const u32x4 w = *reinterpret_cast<const u32x4*>(wl + r * 128 + (((ln % 8) ^ (r & 7)) << 4));
          __builtin_amdgcn_raw_buffer_store_b128(
              w, rc, at < rows && there ? (uint32_t)at * (uint32_t)g.ldc + (uint32_t)(ln % 8 * 16) : kNowhere, 0, 0);
        }
      }
    } else if constexpr (sizeof(OutT) == 2 && EPI != kPlain) {
      // bf16: bias, activation and residual in the lanes as they are, and rows of 64 columns through
      // the slab, u before C. The residual's rows are loaded kDepth slabs ahead.
      constexpr bool kRoom = PITCH == 256;  // the bias has a place behind the slab's rows; else in registers
      constexpr int NH = WTN / 64;
      float* wb = reinterpret_cast<float*>(wl + (kRoom ? 4096 : 0));
#pragma unroll
      for (int k = 0; k < kBias; ++k) wb[k * 64 + ln] = bias1[k];
      f32x4 bias[kRoom ? 1 : FN][4];
      if constexpr (!kRoom) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) bias[j][q] = *reinterpret_cast<const f32x4*>(wb + j * 32 + q * 8 + g4);
      }
      constexpr bool kHasRes = EPI == kEpiRes || EPI == kEpiResKeep;
      constexpr int kSlabs = FM * NH, kDepth = kSlabs < 3 ? kSlabs : 3;
      const int cols = g.N - cur.n0, rows = g.M - cur.m0;
      const void* aux = keeps(EPI) ? g.aux : nullptr;
      const __amdgpu_buffer_rsrc_t rc =
          make_rsrc(uniform(reinterpret_cast<const uint8_t*>(g.C) + ((int64_t)cur.m0 * g.ldc + cur.n0) * 2), kNowhere);
      const __amdgpu_buffer_rsrc_t raux =
          make_rsrc(uniform(reinterpret_cast<const uint8_t*>(aux ? aux : g.C) +
                            (aux ? ((int64_t)cur.m0 * g.ldaux + cur.n0) * 2 : 0)), kNowhere);
      // 32 rows of 64 columns: packed, and out (a piece that N cuts whole: rows hold N rounded up to 8)
      auto put = [&](const uint32_t (&w)[2][8], __amdgpu_buffer_rsrc_t rs, uint32_t ld, int there, int i, int h)
          __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<u32x2*>(wl + fr * 128 + (((j * 4 + q) ^ (fr & 7)) << 4) + g4 * 2) =
                u32x2{w[j][2 * q], w[j][2 * q + 1]};
        u32x4 val[4];
#pragma unroll
        for (int it = 0; it < 4; ++it)
          val[it] = *reinterpret_cast<const u32x4*>(wl + (it * 8 + rr) * 128 + ((gg ^ rr) << 4));
#pragma unroll
        for (int it = 0; it < 4; ++it)
          __builtin_amdgcn_raw_buffer_store_b128(
              val[it], rs, piece_off(ld, there, cols, wm * WTM + i * 32 + it * 8, wn * WTN + h * 64), 0, 2 /* nt */);
      };
      const __amdgpu_buffer_rsrc_t rres =
          make_rsrc(uniform(reinterpret_cast<const uint8_t*>(kHasRes ? g.res : g.C) +
                            (kHasRes ? ((int64_t)cur.m0 * g.ldres + cur.n0) * 2 : 0)), kNowhere);
      u32x4 res[kHasRes ? kDepth : 1][4];
      auto load_res = [&](int s) __attribute__((always_inline)) {
        load_rows(rres, (uint32_t)g.ldres, rows, cols, wm * WTM + s / NH * 32, wn * WTN + s % NH * 64, res[s % kDepth]);
      };
      if constexpr (kHasRes) {
#pragma unroll
        for (int s = 0; s < kDepth; ++s) load_res(s);
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          float v[2][16];
          uint32_t w[2][8];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            asm volatile("" : "+v"(acc[i][h * 2 + j]));  // out of the accumulators here and not before
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              f32x4 b;
              if constexpr (kRoom) b = *reinterpret_cast<const f32x4*>(wb + h * 64 + j * 32 + q * 8 + g4);
              else b = bias[h * 2 + j][q];
#pragma unroll
              for (int k = 0; k < 4; ++k) v[j][4 * q + k] = acc[i][h * 2 + j][4 * q + k] + b[k];
            }
          }
          auto packed = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int k = 0; k < 8; ++k) w[j][k] = pack_bf16x2(v[j][2 * k], v[j][2 * k + 1]);
          };
          if constexpr (keeps(EPI)) {
            packed();
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int k = 0; k < 8; ++k) v[j][2 * k] = bf16_lo(w[j][k]), v[j][2 * k + 1] = bf16_hi(w[j][k]);
            put(w, raux, (uint32_t)g.ldaux, aux ? rows : 0, i, h);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) activate(v[j], g.act);
          if constexpr (kHasRes) {
            const int s = i * NH + h;
            add_rows(res[s % kDepth], v[0], v[1]);
            if (s + kDepth < kSlabs) load_res(s + kDepth);
          }
          packed();
          put(w, rc, (uint32_t)g.ldc, rows, i, h);
        }
    } else if constexpr (EPI != kPlain) {
      // fp32: a lane takes 4 columns of a row (the same ones in every row: its bias stays in registers)
      // from the slab, SC columns at a time, so that residual, u and result are whole rows of pieces.
      constexpr bool kHasRes = EPI == kEpiRes || EPI == kEpiResKeep;
      constexpr int SC = PITCH / 4, NH = WTN / SC;            // NH slabs side by side
      constexpr int LPR = SC / 4, RPI = 64 / LPR, kReads = 32 / RPI, kPieces = SC / 8;
      const int r4 = ln / LPR, c4 = ln % LPR;
      const int cols = g.N - cur.n0, rows = g.M - cur.m0;
      float bias[NH][4];
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k) bias[h][k] = __shfl(bias1[h * SC / 64], h * SC % 64 + c4 * 4 + k, 64);
      auto over_c = [&](const void* p, int64_t ld) __attribute__((always_inline)) {
        return make_rsrc(uniform(reinterpret_cast<const uint8_t*>(p ? p : g.C) + (p ? ((int64_t)cur.m0 * ld + cur.n0) * 4 : 0)),
                         kNowhere);
      };
      const void* aux = keeps(EPI) ? g.aux : nullptr;
      const __amdgpu_buffer_rsrc_t rres = over_c(kHasRes ? g.res : nullptr, g.ldres), raux = over_c(aux, g.ldaux),
                                   rc = over_c(g.C, g.ldc);
      auto at = [&](int64_t ld, int there, int i, int h, int it) __attribute__((always_inline)) {
        const int row = wm * WTM + i * 32 + it * RPI, col = wn * WTN + h * SC;
        return r4 < there - row && c4 * 4 < cols - col ? (((uint32_t)r4 + row) * (uint32_t)ld + c4 * 4 + col) * 4 : kNowhere;
      };
      auto load_res = [&](int s, f32x4 (&r)[kReads]) __attribute__((always_inline)) {
#pragma unroll
        for (int it = 0; it < kReads; ++it)
          r[it] = __builtin_bit_cast(
              f32x4, __builtin_amdgcn_raw_buffer_load_b128(rres, at(g.ldres, rows, s / NH, s % NH, it), 0, 0));
      };
      auto put_slab = [&](int i, int h) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          const int j = h * (SC / 32) + p / 4, q = p % 4;
          if (q == 0) asm volatile("" : "+v"(acc[i][j]));  // out of the accumulators here and not before
          *reinterpret_cast<f32x4*>(wl + fr * PITCH + (((p * 2 + (ln >> 5)) ^ (fr & (LPR - 1))) << 4)) =
              f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        }
      };
      f32x4 res[kHasRes ? 2 : 1][kReads];
      if constexpr (kHasRes) load_res(0, res[0]);
      put_slab(0, 0);
#pragma unroll
      for (int s = 0; s < FM * NH; ++s) {
        const int i = s / NH, h = s % NH;
        if constexpr (kHasRes)
          if (s + 1 < FM * NH) load_res(s + 1, res[(s + 1) & 1]);
        f32x4 x[kReads];
#pragma unroll
        for (int it = 0; it < kReads; ++it) {
          const int r = it * RPI + r4;
          x[it] = *reinterpret_cast<const f32x4*>(wl + r * PITCH + ((c4 ^ (r & (LPR - 1))) << 4));
        }
        if (s + 1 < FM * NH) put_slab((s + 1) / NH, (s + 1) % NH);
#pragma unroll
        for (int it = 0; it < kReads; ++it) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = x[it][k] + bias[h][k];
          if constexpr (keeps(EPI))
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}), raux,
                                                   at(g.ldaux, aux ? rows : 0, i, h, it), 0, 2 /* nt */);
          activate(v, g.act);
          if constexpr (kHasRes) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += res[s & 1][it][k];
          }
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}), rc,
                                                 at(g.ldc, rows, i, h, it), 0, 2 /* nt */);
        }
      }
    } else {
    const bool whole = cur.m0 + BM <= g.M && cur.n0 + BN <= g.N;
    using T = OutT;
    constexpr int SC = PITCH / (int)sizeof(T);                 // columns of a slab
    constexpr int CPR = PITCH / 16, EPC = 16 / (int)sizeof(T), RPI = 64 / CPR;
    constexpr int kSlabs = FM * WTN / SC, kPieces = SC / 8, kReads = 32 / RPI;
    const int r0 = ln / CPR, ch = ln % CPR;
    // piece p of slab s: this lane's 4 columns of 8
    auto piece = [&](int s, int p) __attribute__((always_inline)) {
      const int i = s / (WTN / SC), j = s % (WTN / SC) * (SC / 32) + p / 4, q = p % 4;
      if (q == 0) asm volatile("" : "+v"(acc[i][j]));  // out of the accumulators here and not before
      const int cb = (p * 8 + g4) * (int)sizeof(T);
      uint8_t* at = wl + fr * PITCH + (((cb >> 4) ^ (fr & (CPR - 1))) << 4) + (cb & 15);
      const float x0 = acc[i][j][4 * q], x1 = acc[i][j][4 * q + 1], x2 = acc[i][j][4 * q + 2], x3 = acc[i][j][4 * q + 3];
      if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2*>(at) = u32x2{pack_bf16x2(x0, x1), pack_bf16x2(x2, x3)};
      else *reinterpret_cast<f32x4*>(at) = f32x4{x0, x1, x2, x3};
    };
    auto slab_row = [&](int it) __attribute__((always_inline)) {
      const int r = it * RPI + r0;
      return *reinterpret_cast<const u32x4*>(wl + r * PITCH + ((ch ^ (r & (CPR - 1))) << 4));
    };
    const __amdgpu_buffer_rsrc_t rc =
        make_rsrc(uniform(reinterpret_cast<const uint8_t*>(g.C) + ((int64_t)cur.m0 * g.ldc + cur.n0) * (int64_t)sizeof(T)),
                  kNowhere);
    auto put_whole = [&]() __attribute__((always_inline)) {
      // rows behind one another from a 64-bit base, 32-bit offsets within the tile
      const uint32_t vo = (uint32_t)((r0 * g.ldc + ch * EPC) * (int64_t)sizeof(T));
#pragma unroll
      for (int p = 0; p < kPieces; ++p) piece(0, p);
#pragma unroll
      for (int s = 0; s < kSlabs; ++s) {
        // All of a slab's reads before its first store (the compiler takes a store for one
        // that could change what a later read finds), the next slab's pieces between the
        // stores, which leave 64 bytes a cycle.
        u32x4 val[kReads];
#pragma unroll
        for (int it = 0; it < kReads; ++it) val[it] = slab_row(it);
        const int mrow = wm * WTM + s / (WTN / SC) * 32, ncol = wn * WTN + s % (WTN / SC) * SC;
#pragma unroll
        for (int it = 0; it < kReads; ++it) {
          __builtin_amdgcn_raw_buffer_store_b128(
              val[it], rc, vo, uniform((int)(((mrow + it * RPI) * g.ldc + ncol) * (int64_t)sizeof(T))), 2 /* nt */);
          if (s + 1 < kSlabs) {
#pragma unroll
            for (int p = it * kPieces / kReads; p < (it + 1) * kPieces / kReads; ++p) piece(s + 1, p);
          }
        }
      }
    };
    auto put_edge = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int s = 0; s < kSlabs; ++s) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) piece(s, p);
        // rows and columns past the matrix get an offset out of every range, and a piece
        // that N cuts goes element by element: no lane branches here either
        const int mrow = wm * WTM + s / (WTN / SC) * 32 + r0, ncol = wn * WTN + s % (WTN / SC) * SC + ch * EPC;
        const int n = cur.n0 + ncol;
#pragma unroll 1
        for (int it = 0; it < kReads; ++it) {
          const u32x4 val = slab_row(it);
          const bool in = cur.m0 + mrow + it * RPI < g.M;
          const uint32_t off = (uint32_t)(((mrow + it * RPI) * g.ldc + ncol) * (int64_t)sizeof(T));
          __builtin_amdgcn_raw_buffer_store_b128(val, rc, in && n + EPC <= g.N ? off : kNowhere, 0, 0);
          if (g.N % EPC != 0) {
#pragma unroll
            for (int k = 0; k < EPC - 1; ++k) {
              const uint32_t at = in && n + EPC > g.N && n + k < g.N ? off + k * (uint32_t)sizeof(T) : kNowhere;
              if constexpr (sizeof(T) == 2)
                __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(val[k >> 1] >> (16 * (k & 1))), rc, at, 0, 0);
              else
                __builtin_amdgcn_raw_buffer_store_b32(val[k], rc, at, 0, 0);
            }
          }
        }
      }
    };
    if (g.ws) {
      const __amdgpu_buffer_rsrc_t rw =
          make_rsrc(uniform(reinterpret_cast<const uint8_t*>(g.ws + ((int64_t)cur.split * g.M + cur.m0) * g.ldw + cur.n0)),
                    kNowhere);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = wm * WTM + i * 32 + fr;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          asm volatile("" : "+v"(acc[i][j]));
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int n = wn * WTN + j * 32 + q * 8 + g4;
            const u32x4 v = __builtin_bit_cast(
                u32x4, f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]});
            __builtin_amdgcn_raw_buffer_store_b128(
                v, rw, cur.m0 + m < g.M && cur.n0 + n < g.N ? (uint32_t)((m * g.ldw + n) * 4) : kNowhere, 0, 0);
          }
        }
      }
      wait_vm<0>();
    } else if (whole) {
      // no branch among these stores: the compiler counts them where it lets the next
      // stage's reads pass, and would count none of those it is not sure of
      put_whole();
    } else {
      put_edge();
      wait_vm<0>();
    }
    }
    if (next >= last) wait_vm<0>();  // no DMA is in flight when the workgroup ends
    if (next >= last) break;
    item = next;
    cur = nxt;
  }
}

// C = sum of the splits' partials, in split order; 4 columns a thread.
template <typename OutT>
__global__ __launch_bounds__(256) void f8_reduce_kernel(GemmF8Args g, int splits) {
  const int n = (blockIdx.x * 64 + (threadIdx.x & 63)) * 4;
  if (n >= g.N) return;
  for (int64_t m = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6); m < g.M; m += (int64_t)gridDim.y * 4) {
    const float* p = g.ws + m * g.ldw + n;
    const int64_t step = (int64_t)g.M * g.ldw;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < splits; k0 += 8) {
      f32x4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < splits) v[k] = *reinterpret_cast<const f32x4*>(p + (k0 + k) * step);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < splits) s += v[k];
    }
    OutT* dst = reinterpret_cast<OutT*>(g.C) + m * g.ldc + n;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n + k < g.N) {
        if constexpr (sizeof(OutT) == 2) dst[k] = f32_to_bf16(s[k]);
        else dst[k] = s[k];
      }
  }
}

// The same with an epilogue. Of C in 8 bits a block of 128 is 32 lanes' columns.
template <typename OutT, int EPI>
__global__ __launch_bounds__(256) void f8_reduce_epi_kernel(GemmF8Args g, int splits) {
  using RT = typename std::conditional<sizeof(OutT) == 4, float, uint16_t>::type;  // of residual and u
  const int n = (blockIdx.x * 64 + (threadIdx.x & 63)) * 4;
  if (sizeof(OutT) != 1 && n >= g.N) return;
  auto load4 = [&](const RT* p, float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = 0.f;
      if (n + k < g.N) {
        if constexpr (sizeof(RT) == 2) v[k] = bf16_to_f32(p[k]);
        else v[k] = p[k];
      }
    }
  };
  auto store4 = [&](RT* p, const float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n + k < g.N) {
        if constexpr (sizeof(RT) == 2) p[k] = f32_to_bf16(v[k]);
        else p[k] = v[k];
      }
  };
  float bias[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    bias[k] = 0.f;
    if (g.bias && n + k < g.N)
      bias[k] = g.bias16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(g.bias)[n + k])
                         : reinterpret_cast<const float*>(g.bias)[n + k];
  }
  for (int64_t m = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6); m < g.M; m += (int64_t)gridDim.y * 4) {
    const float* p = g.ws + m * g.ldw + n;
    const int64_t step = (int64_t)g.M * g.ldw;
    float res[4] = {0.f, 0.f, 0.f, 0.f};
    if (g.res) load4(reinterpret_cast<const RT*>(g.res) + m * g.ldres + n, res);
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (n < g.N) {  // (partial rows are whole vectors)
      for (int k0 = 0; k0 < splits; k0 += 8) {
        f32x4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k0 + k < splits) v[k] = *reinterpret_cast<const f32x4*>(p + (k0 + k) * step);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k0 + k < splits) s += v[k];
      }
    }
    float u[4], o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = n + k < g.N ? s[k] + bias[k] : 0.f;
    if constexpr (keeps(EPI)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(RT) == 2) u[k] = bf16_to_f32(f32_to_bf16(u[k]));
        o[k] = u[k];
      }
      if (g.aux) store4(reinterpret_cast<RT*>(g.aux) + m * g.ldaux + n, o);
    }
    activate(u, g.act);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = u[k] + res[k];
    if constexpr (sizeof(OutT) == 1) {
      uint32_t x = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) x = max(x, n + k < g.N ? finite_abs_bits(o[k]) : 0u);
      x = max16(x);
      const auto r16 = __builtin_amdgcn_permlane16_swap(x, x, false, false);
      x = max((uint32_t)r16[0], (uint32_t)r16[1]);
      const int byte = scale_byte(x);
      if (n < (g.N + kB - 1) / kB * kB) {
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = n + k < g.N ? o[k] : 0.f;
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(g.C) + m * g.ldc + n) =
            pack_e4m3x4(o[0], o[1], o[2], o[3], byte);
        if ((threadIdx.x & 31) == 0) g.sc[m * g.ldsc + n / kB] = (uint8_t)byte;
      }
    } else {
      store4(reinterpret_cast<RT*>(g.C) + m * g.ldc + n, o);
    }
  }
}

struct F8Plan {
  bool huge;
  int tiles, splits, kb_chunk;
};

F8Plan f8_plan(int M, int N, int K) {
  const int64_t kb = ((int64_t)K + kB - 1) / kB;
  auto tiles = [&](int t) { return (((int64_t)M + t - 1) / t) * (((int64_t)N + t - 1) / t); };
  F8Plan p;
  // 256 x 256 tiles where there is one for every CU (4096^3 55.8 us against 70.1 with 128 x
  // 128); with 128 of them half the CUs stand idle (16384 x 512 x 2048 26.5 against 22.8,
  // 4096 x 2048 x 2048 25.5 against 19.9). That is measured on tiles that rows fill; the rule
  // counts them however full they are, and 8 x 131072 x 512 takes 22.7 for 14.7, 64 rows 24.7
  // for 16.0.
  p.huge = tiles(256) >= 256;
  const int64_t t = tiles(p.huge ? 256 : 128);
  // A split of K shortens the walk over it (0.39 us a block with a bf16 result, 0.69 with
  // fp32) and costs a second launch (3 us) and its partials written and read (2.6 us per
  // million). Measured (us): 64 x 4096 x 4096 17.2 in one piece, 11.8 in 4, 13.1 in 8; 2048 x
  // 512 x 2048 9.8, 14.4 in 2, 18.8 in 4; 8 x 4096 x 4096 16.0, 8.2 in 8.
  int64_t s = 1, best_s = 1;
  double best = 0.5 * (double)kb;
  if (!p.huge && N <= 1 << 20)  // (a tile's rows of partials within 32-bit offsets)
    for (s = 2; s * t <= 256 && s * 4 <= kb; ++s) {
      const int64_t chunk = ((kb + s - 1) / s + 3) / 4 * 4;
      const double us = 0.5 * (double)chunk + 3.0 + 2.6e-6 * (double)M * (double)N * (double)s;
      if (us < best) best = us, best_s = s;
    }
  s = best_s;
  const int64_t chunk = s > 1 ? ((kb + s - 1) / s + 3) / 4 * 4 : std::max<int64_t>(kb, 1);
  p.splits = (int)std::max<int64_t>(1, (kb + chunk - 1) / chunk);
  p.kb_chunk = (int)chunk;
  p.tiles = t > INT32_MAX ? -1 : (int)t;
  return p;
}

int64_t f8_ldw(int N) { return ((int64_t)N + 3) / 4 * 4; }

template <int BM, int BN, int WTM, int WTN, typename OutT, int EPI, bool kWide = sizeof(OutT) == 4>
void launch_tiles(hipStream_t st, const GemmF8Args& g) {
  const dim3 grid((unsigned)std::min(g.items, (BM * BN >= 65536 ? 1 : 2) * cu_count()));
  if (g.dw) hipLaunchKernelGGL((gemm_f8_kernel<BM, BN, WTM, WTN, OutT, true, EPI, kWide>), grid, dim3(256), 0, st, g);
  else hipLaunchKernelGGL((gemm_f8_kernel<BM, BN, WTM, WTN, OutT, false, EPI, kWide>), grid, dim3(256), 0, st, g);
}

template <typename OutT>
void launch_f8(hipStream_t st, const F8Plan& p, const GemmF8Args& g) {
  if (p.huge) launch_tiles<256, 256, 128, 128, OutT, kPlain>(st, g);
  else launch_tiles<128, 128, 64, 64, OutT, kPlain>(st, g);
  if (p.splits > 1)
    hipLaunchKernelGGL((f8_reduce_kernel<OutT>),
                       dim3((unsigned)((g.N + 255) / 256), (unsigned)std::min<int64_t>(((int64_t)g.M + 3) / 4, 65535)),
                       dim3(256), 0, st, g, p.splits);
}

template <typename OutT, int EPI, bool kWide = sizeof(OutT) == 4>
void launch_f8_epi(hipStream_t st, const F8Plan& p, const GemmF8Args& g) {
  if (p.splits > 1) {
    // partials as the same result without an epilogue has them
    using PT = typename std::conditional<kWide, float, uint16_t>::type;
    launch_tiles<128, 128, 64, 64, PT, kPlain>(st, g);
    hipLaunchKernelGGL((f8_reduce_epi_kernel<OutT, keeps(EPI) ? kEpiKeep : kEpi>),
                       dim3((unsigned)((g.N + 255) / 256), (unsigned)std::min<int64_t>(((int64_t)g.M + 3) / 4, 65535)),
                       dim3(256), 0, st, g, p.splits);
  } else if (p.huge) {
    launch_tiles<256, 256, 128, 128, OutT, EPI, kWide>(st, g);
  } else if constexpr (sizeof(OutT) == 1) {
    launch_tiles<128, 128, 32, 128, OutT, EPI>(st, g);
  } else {
    launch_tiles<128, 128, 64, 64, OutT, EPI, kWide>(st, g);
  }
}

// 256 rows of a tile are addressed with 31-bit offsets: bytes of an operand's row, elements of a result's
constexpr int64_t kMaxLd = INT32_MAX / 256, kMaxLdc = INT32_MAX / 256 / 4;

// The checks of one quantised operand: rows x K, group rows per scale.
int check_operand(const char* what, int64_t rows, int64_t K, const void* q, int64_t ld, const void* s, int64_t lds,
                  int group) {
  const int64_t kb = (K + kB - 1) / kB;
  if (group != 1 && group != kB) return nl_set_error(NL_EINVAL, std::string(what) + ": a scale holds for 1 or 128 rows");
  if (rows == 0 || K == 0) return NL_OK;
  if (!q || !s) return nl_set_error(NL_EINVAL, std::string(what) + ": null pointer");
  if (ld < kb * kB) return nl_set_error(NL_EINVAL, std::string(what) + ": rows hold whole blocks of 128 (leading dimension)");
  if (lds < kb) return nl_set_error(NL_EINVAL, std::string(what) + ": a scale row is shorter than its blocks");
  if (ld % 16 || ((uintptr_t)q & 15))
    return nl_set_error(NL_EALIGN, std::string(what) + ": values need 16-byte aligned rows");
  return NL_OK;
}

}  // namespace
}  // namespace nl

using namespace nl;

namespace nl {
namespace {

// The checks of nl_quantize_fp8, and its kernel's arguments (rows or cols 0: nothing to do).
// sums: what is written is the column sums (too).
int quant_args(int64_t rows, int64_t cols, const void* x, int x_dtype, int64_t ldx, int group, uint8_t* q, int64_t ldq,
               uint8_t* scale, int64_t lds, uint8_t* qt, int64_t ldqt, uint8_t* scale_t, int64_t ldst, QuantArgs* out,
               bool sums = false) {
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > INT32_MAX)
    return nl_set_error(NL_EINVAL, "quantize_fp8: need 0 <= rows, cols < 2^31");
  if (x_dtype != NL_DTYPE_F32 && x_dtype != NL_DTYPE_BF16)
    return nl_set_error(NL_EINVAL, "quantize_fp8: x is fp32 or bf16");
  if (!q && !qt && !sums) return nl_set_error(NL_EINVAL, "quantize_fp8: no output");
  if (q)
    if (int rc = check_operand("quantize_fp8", rows, cols, q, ldq, scale, lds, group)) return rc;
  if (qt)
    if (int rc = check_operand("quantize_fp8 (transpose)", cols, rows, qt, ldqt, scale_t, ldst, group)) return rc;
  if (rows == 0 || cols == 0) return NL_OK;
  const int esz = x_dtype == NL_DTYPE_BF16 ? 2 : 4;
  if (!x) return nl_set_error(NL_EINVAL, "quantize_fp8: null x");
  if (rows > 1 && ldx < cols) return nl_set_error(NL_EINVAL, "quantize_fp8: ldx < cols");
  if ((uintptr_t)x % esz) return nl_set_error(NL_EALIGN, "quantize_fp8: x is not aligned to its type");
  *out = QuantArgs{rows, cols, x, ldx, group, q, ldq, scale, lds, qt, ldqt, scale_t, ldst};
  return NL_OK;
}

// The same of dy * act'(u), with its column sums: dbias, over partial rows in ws.
int dact_args(int64_t rows, int64_t cols, const void* dy, int dtype, int64_t lddy, const void* u, int64_t ldu, int act,
              uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds, uint8_t* qt, int64_t ldqt, uint8_t* scale_t,
              int64_t ldst, const void* dbias, int db_dtype, float* part, QuantArgs* out) {
  const char* what = "quantize_fp8_dact";
  if (act < NL_ACT_NONE || act > NL_ACT_SILU) return nl_set_error(NL_EINVAL, std::string(what) + ": unknown activation");
  if (int rc = quant_args(rows, cols, dy, dtype, lddy, 1, q, ldq, scale, lds, qt, ldqt, scale_t, ldst, out,
                          dbias != nullptr))
    return rc;
  if (dbias && cols > 1 << 25) return nl_set_error(NL_EUNSUPPORTED, std::string(what) + ": a bias of more than 2^25");
  if (rows == 0 || cols == 0) return NL_OK;
  if (act != NL_ACT_NONE) {
    const int esz = dtype == NL_DTYPE_BF16 ? 2 : 4;
    if (!u) return nl_set_error(NL_EINVAL, std::string(what) + ": null u");
    if (rows > 1 && ldu < cols) return nl_set_error(NL_EINVAL, std::string(what) + ": ldu < cols");
    if ((uintptr_t)u % esz) return nl_set_error(NL_EALIGN, std::string(what) + ": u is not aligned to its type");
  }
  if (dbias && !part) return nl_set_error(NL_EINVAL, std::string(what) + ": workspace too small");
  if (dbias && db_dtype != NL_DTYPE_F32 && db_dtype != NL_DTYPE_BF16)
    return nl_set_error(NL_EINVAL, std::string(what) + ": dbias is fp32 or bf16");
  if ((uintptr_t)dbias & (db_dtype == NL_DTYPE_BF16 ? 1 : 3))
    return nl_set_error(NL_EALIGN, std::string(what) + ": dbias is not aligned to its type");
  out->u = u, out->ldu = ldu, out->act = act, out->part = dbias ? part : nullptr;
  return NL_OK;
}

int64_t blocks_of(int64_t n) { return (n + kB - 1) / kB; }
// a launch has fewer than 2^32 threads: 16 a block of 128 by rows in whole groups of 256, 512 a tile
constexpr int64_t kMaxBlocks = ((int64_t)1 << 28) - 16, kMaxTiles = ((int64_t)1 << 23) - 1;

template <bool kAct>
int quantize_one(hipStream_t st, const QuantArgs& a, int dtype) {
  const int64_t rb = blocks_of(a.rows), cb = blocks_of(a.cols);
  if (!a.qt && a.group == 1 && !a.part) {
    const int64_t blocks = a.rows * cb;
    if (blocks > kMaxBlocks) return nl_set_error(NL_EUNSUPPORTED, "quantize_fp8: more than 2^28 - 16 blocks");
    const dim3 grid((unsigned)((blocks + 15) / 16));
    if (dtype == NL_DTYPE_BF16)
      hipLaunchKernelGGL((quantize_rows_kernel<uint16_t, kAct>), grid, dim3(256), 0, st, a, (uint32_t)blocks, (uint32_t)cb);
    else
      hipLaunchKernelGGL((quantize_rows_kernel<float, kAct>), grid, dim3(256), 0, st, a, (uint32_t)blocks, (uint32_t)cb);
    return nl_check_launch("nl_quantize_fp8");
  }
  if (rb * cb > kMaxTiles) return nl_set_error(NL_EUNSUPPORTED, "quantize_fp8: 2^23 tiles of 128 x 128 and more");
  const dim3 grid((unsigned)(rb * cb));
  if (dtype == NL_DTYPE_BF16)
    hipLaunchKernelGGL((quantize_tile_kernel<uint16_t, kAct>), grid, dim3(512), 0, st, a, (uint32_t)cb);
  else
    hipLaunchKernelGGL((quantize_tile_kernel<float, kAct>), grid, dim3(512), 0, st, a, (uint32_t)cb);
  return nl_check_launch("nl_quantize_fp8");
}

// Two matrices in one launch where both go by tiles (and there is room for the grid).
int quantize_two(hipStream_t st, const QuantArgs& a, int a_dtype, const QuantArgs& b, int b_dtype) {
  const int64_t ca = blocks_of(a.cols), cb = blocks_of(b.cols);
  const int64_t na = blocks_of(a.rows) * ca, nb = blocks_of(b.rows) * cb;
  if ((!a.qt && a.group == 1) || (!b.qt && b.group == 1) || na + nb > kMaxTiles) {
    if (int rc = quantize_one<false>(st, a, a_dtype)) return rc;
    return quantize_one<false>(st, b, b_dtype);
  }
  const dim3 grid((unsigned)(na + nb));
#define NL_QUANT_TWO(TA, TB)                                                                                  \
  hipLaunchKernelGGL((quantize_two_kernel<TA, TB>), grid, dim3(512), 0, st, a, (uint32_t)ca, (uint32_t)na, b, \
                     (uint32_t)cb)
  if (a_dtype == NL_DTYPE_BF16) {
    if (b_dtype == NL_DTYPE_BF16) NL_QUANT_TWO(uint16_t, uint16_t);
    else NL_QUANT_TWO(uint16_t, float);
  } else {
    if (b_dtype == NL_DTYPE_BF16) NL_QUANT_TWO(float, uint16_t);
    else NL_QUANT_TWO(float, float);
  }
#undef NL_QUANT_TWO
  return nl_check_launch("nl_quantize_fp8");
}

}  // namespace
}  // namespace nl

extern "C" int nl_quantize_fp8(void* stream, int64_t rows, int64_t cols, const void* x, int x_dtype, int64_t ldx,
                               int group, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds, uint8_t* qt,
                               int64_t ldqt, uint8_t* scale_t, int64_t ldst) {
  QuantArgs a;
  if (int rc = quant_args(rows, cols, x, x_dtype, ldx, group, q, ldq, scale, lds, qt, ldqt, scale_t, ldst, &a))
    return rc;
  return rows == 0 || cols == 0 ? NL_OK : quantize_one<false>((hipStream_t)stream, a, x_dtype);
}

namespace nl {
namespace {

int quantize_dact(hipStream_t st, const QuantArgs& a, int dtype, void* dbias, int db_dtype) {
  const int rc = a.act == NL_ACT_NONE && !a.part ? quantize_one<false>(st, a, dtype) : quantize_one<true>(st, a, dtype);
  if (rc || !a.part) return rc;
  launch_partial_sums(st, (int)blocks_of(a.rows), (int)a.cols, a.part, dbias, db_dtype, 0);
  return nl_check_launch("nl_quantize_fp8_dact");
}

}  // namespace
}  // namespace nl

extern "C" size_t nl_quantize_fp8_dact_ws_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : (size_t)blocks_of(rows) * cols * sizeof(float);
}

extern "C" int nl_quantize_fp8_dact(void* stream, int64_t rows, int64_t cols, const void* dy, int dtype, int64_t lddy,
                                    const void* u, int64_t ldu, int act, uint8_t* q, int64_t ldq, uint8_t* scale,
                                    int64_t lds, uint8_t* qt, int64_t ldqt, uint8_t* scale_t, int64_t ldst,
                                    void* dbias, int db_dtype, void* ws, size_t ws_bytes) {
  QuantArgs a;
  if ((uintptr_t)ws & 3) return nl_set_error(NL_EALIGN, "quantize_fp8_dact: workspace not aligned");
  float* part = ws && ws_bytes >= nl_quantize_fp8_dact_ws_bytes(rows, cols) ? (float*)ws : nullptr;
  if (int rc = dact_args(rows, cols, dy, dtype, lddy, u, ldu, act, q, ldq, scale, lds, qt, ldqt, scale_t, ldst, dbias,
                         db_dtype, part, &a))
    return rc;
  if (cols == 0 || (rows == 0 && !dbias)) return NL_OK;
  if (rows == 0) {
    launch_partial_sums((hipStream_t)stream, 0, (int)cols, part, dbias, db_dtype, 0);
    return nl_check_launch("nl_quantize_fp8_dact");
  }
  return quantize_dact((hipStream_t)stream, a, dtype, dbias, db_dtype);
}

extern "C" size_t nl_gemm_fp8_ws_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const F8Plan p = f8_plan(M, N, K);
  return p.splits > 1 ? (size_t)p.splits * M * f8_ldw(N) * sizeof(float) : 0;
}

namespace nl {
namespace {

// The epilogue of a product as its callers give it; none: all as below.
struct F8Epilogue {
  int kind = kPlain;
  const void* bias = nullptr;
  int bias_dtype = NL_DTYPE_F32;
  int act = NL_ACT_NONE;
  const void* res = nullptr;
  int64_t ldres = 0;
  void* aux = nullptr;
  int64_t ldaux = 0;
  uint8_t* sc = nullptr;
  int64_t ldsc = 0;
};

// A matrix over C of the epilogue's: rows that 16-byte pieces divide.
int check_over_c(const char* name, const void* p, int64_t ld, int N) {
  if (!p) return NL_OK;
  if (ld < N) return nl_set_error(NL_EINVAL, std::string("gemm_fp8: rows of ") + name + " are shorter than N");
  if (((uintptr_t)p & 15) || ld % 8)
    return nl_set_error(NL_EALIGN, std::string("gemm_fp8: ") + name + " needs 16-byte aligned rows");
  if (ld > kMaxLdc) return nl_set_error(NL_EUNSUPPORTED, std::string("gemm_fp8: rows of ") + name + " of 2 million elements and more");
  return NL_OK;
}

int gemm_fp8(void* stream, int M, int N, int K, const uint8_t* A, int64_t lda, const uint8_t* scale_a, int64_t ldsa,
             int group_a, const uint8_t* B, int64_t ldb, const uint8_t* scale_b, int64_t ldsb, int group_b, void* C,
             int c_dtype, int64_t ldc, const F8Epilogue& e, void* ws, size_t ws_bytes) {
  if (M < 0 || N < 0 || K < 0) return nl_set_error(NL_EINVAL, "gemm_fp8: need M, N, K >= 0");
  const bool c8 = c_dtype == NL_DTYPE_E4M3;
  if (c_dtype != NL_DTYPE_F32 && c_dtype != NL_DTYPE_BF16 && !(c8 && e.kind != kPlain))
    return nl_set_error(NL_EINVAL, "gemm_fp8: C is fp32 or bf16");
  if (e.act < NL_ACT_NONE || e.act > NL_ACT_SILU) return nl_set_error(NL_EINVAL, "gemm_fp8: unknown activation");
  if (int rc = check_operand("gemm_fp8 A", M, K, A, lda, scale_a, ldsa, group_a)) return rc;
  if (int rc = check_operand("gemm_fp8 B", N, K, B, ldb, scale_b, ldsb, group_b)) return rc;
  if (M == 0 || N == 0) return NL_OK;
  if (!C) return nl_set_error(NL_EINVAL, "gemm_fp8: null C");
  if (c8) {
    if (e.aux) return nl_set_error(NL_EINVAL, "gemm_fp8: a result in 8 bits keeps no u");
    if (int rc = check_operand("gemm_fp8 C", M, N, C, ldc, e.sc, e.ldsc, 1)) return rc;
  } else {
    if (ldc < N) return nl_set_error(NL_EINVAL, "gemm_fp8: ldc < N");
    if (((uintptr_t)C & 15) || ldc % 8) return nl_set_error(NL_EALIGN, "gemm_fp8: C needs 16-byte aligned rows");
  }
  if (e.bias && e.bias_dtype != NL_DTYPE_F32 && e.bias_dtype != NL_DTYPE_BF16)
    return nl_set_error(NL_EINVAL, "gemm_fp8: bias is fp32 or bf16");
  const int bias16 = e.bias_dtype == NL_DTYPE_BF16 ? 1 : 0;
  if ((uintptr_t)e.bias & (bias16 ? 1 : 3)) return nl_set_error(NL_EALIGN, "gemm_fp8: bias is not aligned to its type");
  if (int rc = check_over_c("the residual", e.res, e.ldres, N)) return rc;
  if (int rc = check_over_c("aux", e.aux, e.ldaux, N)) return rc;
  const int64_t Kp = ((int64_t)K + kB - 1) / kB * kB;
  if (ldc > kMaxLdc) return nl_set_error(NL_EUNSUPPORTED, "gemm_fp8: rows of C of 2 million elements and more");
  if (lda > kMaxLd || ldb > kMaxLd || ldsa > kMaxLd || ldsb > kMaxLd)
    return nl_set_error(NL_EUNSUPPORTED, "gemm_fp8: rows of 8 MiB and more");
  F8Plan p = f8_plan(M, N, K);
  // relu in front of a backward pass: the sign of u decides whether a gradient passes, and sums cut at
  // 2^-13 of a product had it wrong for one u in 100000 (an error of 0.6% in dx): fp32 sums, whatever
  // the result's type. That costs a layer's forward (us, with its quantisers) 60 for 52 with gelu's sums
  // at 16384 x 512 x 2048, 142 for 92 at 4096^3; with 256 x 256 tiles 66 and 144. It is paid where no gradient
  // is wanted, too: a layer's output does not depend on that.
  // A result in 8 bits is summed with the cut. Of normal operands it leaves 9e-4 of the bytes a step beside
  // those of fp32 sums: 9e-4 of the result's norm, where the rounding to 8 bits is 2.7e-2. With fp32 sums (us, gelu):
  // 16384 x 2048 x 512 49 for 34, 16384 x 512 x 2048 36 for 23, 16384 x 8192 x 1024 275 for 170, 8192^3 760 for 415.
  const bool fine = c_dtype == NL_DTYPE_F32 || (e.kind == kEpiKeep && e.act == NL_ACT_RELU);
  // 128 x 128 tiles, two workgroups a CU, where the epilogue of one runs beside the other's walk over a
  // short K, although each operand is read twice as often. Measured (us, against 256 x 256): C in 8 bits
  // with gelu 16384 x 2048 x 512 33.2 and 39.2, 16384 x 8192 x 1024 169 and 183, 16384 x 2048 x 2048 72.5
  // and 72.1, with a residual 82 and 89; u kept 41.8 and 49.5, 204 and 214, 82.6 and 83.2, 4096^3 77 and
  // 65; a residual alone 36.3 and 40.0, 218 and 216; neither 33.6 and 34.4, 174 and 164.
  const int64_t shallow = c8 ? (e.res ? 2048 : 1024) : e.kind == kEpiKeep && e.aux ? 2048 : e.res ? 512 : 0;
  if (e.kind != kPlain && p.huge && Kp <= shallow) {
    p.huge = false;
    const int64_t t = (((int64_t)M + 127) / 128) * (((int64_t)N + 127) / 128);
    p.tiles = t > INT32_MAX ? -1 : (int)t;
  }
  if (p.tiles < 0 || (int64_t)p.tiles * p.splits > INT32_MAX) return nl_set_error(NL_EUNSUPPORTED, "gemm_fp8: too many tiles");
  auto dwords = [](const void* s, int64_t ld) { return ld % 4 == 0 && ((uintptr_t)s & 3) == 0; };
  GemmF8Args g{M, N, K, (int)Kp,
               A, lda, scale_a, ldsa, group_a == kB ? 7 : 0,
               B, ldb, scale_b, ldsb, group_b == kB ? 7 : 0,
               dwords(scale_a, ldsa) && dwords(scale_b, ldsb) ? 1 : 0,
               C, ldc, nullptr, f8_ldw(N), p.tiles, 0, p.kb_chunk,
               e.bias, bias16, e.act, e.res, e.ldres, e.aux, e.ldaux, e.sc, e.ldsc};
  if (p.splits > 1) {
    if (ws && ws_bytes >= nl_gemm_fp8_ws_bytes(M, N, K)) {
      if ((uintptr_t)ws & 15) return nl_set_error(NL_EALIGN, "gemm_fp8: workspace not 16-byte aligned");
      g.ws = (float*)ws;
    } else {
      p.splits = 1;
      g.kb_chunk = (int)(Kp / kB);
    }
  }
  g.items = p.tiles * p.splits;
  const hipStream_t st = (hipStream_t)stream;
  if (e.kind == kPlain) {
    if (c_dtype == NL_DTYPE_F32) launch_f8<float>(st, p, g);
    else launch_f8<uint16_t>(st, p, g);
  } else if (c8) {
    e.res ? launch_f8_epi<uint8_t, kEpiRes>(st, p, g) : launch_f8_epi<uint8_t, kEpi>(st, p, g);
  } else if (c_dtype == NL_DTYPE_F32) {  // (in fp32 u is not rounded)
    if (e.aux) e.res ? launch_f8_epi<float, kEpiResKeep>(st, p, g) : launch_f8_epi<float, kEpiKeep>(st, p, g);
    else e.res ? launch_f8_epi<float, kEpiRes>(st, p, g) : launch_f8_epi<float, kEpi>(st, p, g);
  } else {
    if (fine) e.res ? launch_f8_epi<uint16_t, kEpiResKeep, true>(st, p, g) : launch_f8_epi<uint16_t, kEpiKeep, true>(st, p, g);
    else if (e.kind == kEpiKeep) e.res ? launch_f8_epi<uint16_t, kEpiResKeep>(st, p, g) : launch_f8_epi<uint16_t, kEpiKeep>(st, p, g);
    else e.res ? launch_f8_epi<uint16_t, kEpiRes>(st, p, g) : launch_f8_epi<uint16_t, kEpi>(st, p, g);
  }
  return nl_check_launch("nl_gemm_fp8");
}

}  // namespace
}  // namespace nl

extern "C" int nl_gemm_fp8(void* stream, int M, int N, int K, const uint8_t* A, int64_t lda, const uint8_t* scale_a,
                           int64_t ldsa, int group_a, const uint8_t* B, int64_t ldb, const uint8_t* scale_b,
                           int64_t ldsb, int group_b, void* C, int c_dtype, int64_t ldc, void* ws, size_t ws_bytes) {
  return gemm_fp8(stream, M, N, K, A, lda, scale_a, ldsa, group_a, B, ldb, scale_b, ldsb, group_b, C, c_dtype, ldc,
                  F8Epilogue{}, ws, ws_bytes);
}

extern "C" int nl_gemm_fp8_fused(void* stream, int M, int N, int K, const uint8_t* A, int64_t lda,
                                 const uint8_t* scale_a, int64_t ldsa, int group_a, const uint8_t* B, int64_t ldb,
                                 const uint8_t* scale_b, int64_t ldsb, int group_b, const void* bias, int bias_dtype,
                                 int act, const void* residual, int64_t ldr, int round_u, void* aux, int64_t ldaux, void* C,
                                 int c_dtype, int64_t ldc, uint8_t* scale_c, int64_t ldsc, void* ws, size_t ws_bytes) {
  F8Epilogue e;
  e.kind = round_u || aux ? kEpiKeep : kEpi;
  e.bias = bias, e.bias_dtype = bias_dtype, e.act = act, e.res = residual, e.ldres = ldr, e.aux = aux, e.ldaux = ldaux;
  e.sc = scale_c, e.ldsc = ldsc;
  if (c_dtype == NL_DTYPE_E4M3 && round_u) return nl_set_error(NL_EINVAL, "gemm_fp8: a result in 8 bits does not round u");
  return gemm_fp8(stream, M, N, K, A, lda, scale_a, ldsa, group_a, B, ldb, scale_b, ldsb, group_b, C, c_dtype, ldc, e,
                  ws, ws_bytes);
}

// ===========================================================================
// linear and its gradients in one call each
// ===========================================================================
namespace nl {
namespace {

// A quantised operand inside a byte buffer: values, then scale rows of whole dwords.
struct Part {
  int64_t rows, cols;  // cols: the summed axis
  int group;
  int64_t at = 0, sat = 0;
  int64_t ld() const { return (cols + kB - 1) / kB * kB; }
  int64_t lds() const { return ((cols + kB - 1) / kB + 3) / 4 * 4; }
  // places it at `end` (a multiple of 16) and returns the end behind it
  int64_t place(int64_t end) {
    at = end;
    sat = at + rows * ld();
    return (sat + (rows + group - 1) / group * lds() + 15) / 16 * 16;
  }
};

struct LinearParts {
  Part wb, xt;      // kept for the gradients: W (K, N), X^T (K, M)
  Part x, wf;       // of the forward: X (M, K), W^T (N, K)
  Part dy, dyt;     // of the backward: dY (M, N), dY^T (N, M)
  int64_t saved, fwd, bwd;
  size_t ws_fwd, ws_dx, ws_dw;
};

LinearParts linear_parts(int M, int K, int N, bool dx, bool dw) {
  LinearParts p{};
  p.wb = {K, N, kB};
  p.xt = {K, M, 1};
  p.x = {M, K, 1};
  p.wf = {N, K, kB};
  p.dy = {M, N, 1};
  p.dyt = {N, M, 1};
  if (dx) p.saved = p.wb.place(p.saved);
  if (dw) p.saved = p.xt.place(p.saved);
  p.fwd = p.wf.place(p.x.place(0));
  if (dx) p.bwd = p.dy.place(p.bwd);
  if (dw) p.bwd = p.dyt.place(p.bwd);
  p.ws_fwd = nl_gemm_fp8_ws_bytes(M, N, K);
  p.ws_dx = dx ? nl_gemm_fp8_ws_bytes(M, K, N) : 0;
  p.ws_dw = dw ? nl_gemm_fp8_ws_bytes(K, N, M) : 0;
  return p;
}

int part_args(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t cols, uint8_t* buf, const Part* a,
              uint8_t* tbuf, const Part* t, QuantArgs* out) {
  return quant_args(rows, cols, x, dtype, ldx, a ? a->group : t->group, a ? buf + a->at : nullptr, a ? a->ld() : 0,
                    a ? buf + a->sat : nullptr, a ? a->lds() : 0, t ? tbuf + t->at : nullptr, t ? t->ld() : 0,
                    t ? tbuf + t->sat : nullptr, t ? t->lds() : 0, out);
}

int product(void* st, const uint8_t* abuf, const Part& a, const uint8_t* bbuf, const Part& b, void* C, int dtype,
            int64_t ldc, void* ws, size_t wsb, const F8Epilogue& e = F8Epilogue{}) {
  return gemm_fp8(st, (int)a.rows, (int)b.rows, (int)a.cols, abuf + a.at, a.ld(), abuf + a.sat, a.lds(), a.group,
                  bbuf + b.at, b.ld(), bbuf + b.sat, b.lds(), b.group, C, dtype, ldc, e, wsb ? ws : nullptr, wsb);
}

int check_linear(const char* what, int M, int K, int N, const void* buf, size_t have, int64_t want, const char* name) {
  if (M < 0 || K < 0 || N < 0) return nl_set_error(NL_EINVAL, std::string(what) + ": need M, K, N >= 0");
  if (want > 0 && (!buf || have < (size_t)want))
    return nl_set_error(NL_EINVAL, std::string(what) + ": " + name + " too small");
  if ((uintptr_t)buf & 15) return nl_set_error(NL_EALIGN, std::string(what) + ": " + name + " not 16-byte aligned");
  return NL_OK;
}

// What the backward of a forward pass would refuse is refused before it: X^T's rows of M bytes,
// dX's of K elements (128 columns of padding at most), dY by rows.
int check_gradients(int M, int K, int N, bool dx, bool dw) {
  if (dw && blocks_of(M) * kB > kMaxLd)
    return nl_set_error(NL_EUNSUPPORTED, "linear_fp8_fwd: a weight gradient over more than 8388480 rows");
  if (dx && K > kMaxLdc - kB)
    return nl_set_error(NL_EUNSUPPORTED, "linear_fp8_fwd: an input gradient of more than 2 million columns");
  if (dx && !dw && M * blocks_of(N) > kMaxBlocks)
    return nl_set_error(NL_EUNSUPPORTED, "linear_fp8_fwd: an output gradient of more than 2^28 - 16 blocks");
  return NL_OK;
}

}  // namespace
}  // namespace nl

extern "C" size_t nl_linear_fp8_saved_bytes(int M, int K, int N, int need_dx, int need_dw) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  return (size_t)linear_parts(M, K, N, need_dx != 0, need_dw != 0).saved;
}

extern "C" size_t nl_linear_fp8_ws_bytes(int M, int K, int N, int backward, int need_dx, int need_dw) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  const LinearParts p = linear_parts(M, K, N, need_dx != 0, need_dw != 0);
  return backward ? (size_t)p.bwd + std::max(p.ws_dx, p.ws_dw) : (size_t)p.fwd + p.ws_fwd;
}

namespace nl {
namespace {

int linear_fwd(void* stream, int M, int K, int N, const void* x, int x_dtype, int64_t ldx, const void* W, int w_dtype,
               int64_t ldw, const F8Epilogue& e, void* y, int y_dtype, int64_t ldy, int need_dx, int need_dw,
               void* saved, size_t saved_bytes, void* ws, size_t ws_bytes) {
  if (M <= 0 || K <= 0 || N <= 0) return nl_set_error(NL_EINVAL, "linear_fp8_fwd: need M, K, N > 0");
  if (int rc = check_gradients(M, K, N, need_dx != 0, need_dw != 0)) return rc;
  const LinearParts p = linear_parts(M, K, N, need_dx != 0, need_dw != 0);
  if (int rc = check_linear("linear_fp8_fwd", M, K, N, saved, saved_bytes, p.saved, "saved buffer")) return rc;
  if (int rc = check_linear("linear_fp8_fwd", M, K, N, ws, ws_bytes, p.fwd + (int64_t)p.ws_fwd, "workspace")) return rc;
  uint8_t *sv = (uint8_t*)saved, *b = (uint8_t*)ws;
  QuantArgs qw, qx;
  if (int rc = part_args(W, w_dtype, ldw, K, N, sv, need_dx ? &p.wb : nullptr, b, &p.wf, &qw)) return rc;
  if (int rc = part_args(x, x_dtype, ldx, M, K, b, &p.x, sv, need_dw ? &p.xt : nullptr, &qx)) return rc;
  if (int rc = quantize_two((hipStream_t)stream, qx, x_dtype, qw, w_dtype)) return rc;
  return product(stream, b, p.x, b, p.wf, y, y_dtype, ldy, b + p.fwd, p.ws_fwd, e);
}

// dy * act'(u) quantised for the wanted gradients; dbias (may be null) over partial rows behind
// what else the workspace holds.
int linear_bwd(void* stream, int M, int K, int N, const void* dy, int dy_dtype, int64_t lddy, const void* u,
               int64_t ldu, int act, void* dbias, int db_dtype, const void* saved, size_t saved_bytes, int need_dx, int need_dw,
               void* dx, int dx_dtype, int64_t lddx, void* dW, int dw_dtype, int64_t lddw, void* ws, size_t ws_bytes) {
  if (M <= 0 || K <= 0 || N <= 0) return nl_set_error(NL_EINVAL, "linear_fp8_bwd: need M, K, N > 0");
  if (!need_dx && !need_dw && !dbias) return NL_OK;
  const LinearParts p = linear_parts(M, K, N, need_dx != 0, need_dw != 0);
  const int64_t behind = p.bwd + (int64_t)std::max(p.ws_dx, p.ws_dw);
  const int64_t sums = dbias ? (int64_t)nl_quantize_fp8_dact_ws_bytes(M, N) : 0;
  if (int rc = check_linear("linear_fp8_bwd", M, K, N, saved, saved_bytes, p.saved, "saved buffer")) return rc;
  if (int rc = check_linear("linear_fp8_bwd", M, K, N, ws, ws_bytes, behind + sums, "workspace")) return rc;
  const uint8_t* sv = (const uint8_t*)saved;
  uint8_t* b = (uint8_t*)ws;
  QuantArgs q;
  if (int rc = dact_args(M, N, dy, dy_dtype, lddy, u, ldu, act, need_dx ? b + p.dy.at : nullptr, p.dy.ld(),
                         need_dx ? b + p.dy.sat : nullptr, p.dy.lds(), need_dw ? b + p.dyt.at : nullptr, p.dyt.ld(),
                         need_dw ? b + p.dyt.sat : nullptr, p.dyt.lds(), dbias, db_dtype, (float*)(b + behind), &q))
    return rc;
  if (int rc = quantize_dact((hipStream_t)stream, q, dy_dtype, dbias, db_dtype)) return rc;
  if (need_dx)
    if (int rc = product(stream, b, p.dy, sv, p.wb, dx, dx_dtype, lddx, b + p.bwd, p.ws_dx)) return rc;
  if (need_dw)
    if (int rc = product(stream, sv, p.xt, b, p.dyt, dW, dw_dtype, lddw, b + p.bwd, p.ws_dw)) return rc;
  return NL_OK;
}

}  // namespace
}  // namespace nl

extern "C" int nl_linear_fp8_fwd(void* stream, int M, int K, int N, const void* x, int x_dtype, int64_t ldx,
                                 const void* W, int w_dtype, int64_t ldw, void* y, int y_dtype, int64_t ldy,
                                 int need_dx, int need_dw, void* saved, size_t saved_bytes, void* ws,
                                 size_t ws_bytes) {
  return linear_fwd(stream, M, K, N, x, x_dtype, ldx, W, w_dtype, ldw, F8Epilogue{}, y, y_dtype, ldy, need_dx, need_dw,
                    saved, saved_bytes, ws, ws_bytes);
}

extern "C" int nl_linear_fp8_bwd(void* stream, int M, int K, int N, const void* dy, int dy_dtype, int64_t lddy,
                                 const void* saved, size_t saved_bytes, int need_dx, int need_dw, void* dx,
                                 int dx_dtype, int64_t lddx, void* dW, int dw_dtype, int64_t lddw, void* ws,
                                 size_t ws_bytes) {
  return linear_bwd(stream, M, K, N, dy, dy_dtype, lddy, nullptr, 0, NL_ACT_NONE, nullptr, 0, saved, saved_bytes, need_dx,
                    need_dw, dx, dx_dtype, lddx, dW, dw_dtype, lddw, ws, ws_bytes);
}

extern "C" size_t nl_linear_fp8_fused_ws_bytes(int M, int K, int N, int backward, int need_dx, int need_dw,
                                               int need_db) {
  return nl_linear_fp8_ws_bytes(M, K, N, backward, need_dx, need_dw) +
         (backward && need_db ? nl_quantize_fp8_dact_ws_bytes(M, N) : 0);
}

extern "C" int nl_linear_fp8_fused_fwd(void* stream, int M, int K, int N, const void* x, int x_dtype, int64_t ldx,
                                       const void* W, int w_dtype, int64_t ldw, const void* bias, int bias_dtype,
                                       int act, const void* residual, int64_t ldr, void* u, int64_t ldu, void* y, int y_dtype,
                                       int64_t ldy, int need_dx, int need_dw, void* saved, size_t saved_bytes,
                                       void* ws, size_t ws_bytes) {
  F8Epilogue e;
  e.kind = act != NL_ACT_NONE ? kEpiKeep : kEpi;
  e.bias = bias, e.bias_dtype = bias_dtype, e.act = act, e.res = residual, e.ldres = ldr;
  e.aux = act != NL_ACT_NONE ? u : nullptr, e.ldaux = ldu;
  return linear_fwd(stream, M, K, N, x, x_dtype, ldx, W, w_dtype, ldw, e, y, y_dtype, ldy, need_dx, need_dw, saved,
                    saved_bytes, ws, ws_bytes);
}

extern "C" int nl_linear_fp8_fused_bwd(void* stream, int M, int K, int N, const void* dy, int dy_dtype, int64_t lddy,
                                       const void* u, int64_t ldu, int act, void* dbias, int db_dtype,
                                       const void* saved, size_t saved_bytes, int need_dx, int need_dw, void* dx, int dx_dtype,
                                       int64_t lddx, void* dW, int dw_dtype, int64_t lddw, void* ws, size_t ws_bytes) {
  return linear_bwd(stream, M, K, N, dy, dy_dtype, lddy, u, ldu, act, dbias, db_dtype, saved, saved_bytes, need_dx, need_dw, dx,
                    dx_dtype, lddx, dW, dw_dtype, lddw, ws, ws_bytes);
}
