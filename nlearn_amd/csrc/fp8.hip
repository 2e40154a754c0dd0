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

#include "common.h"

namespace nl {
namespace {

constexpr int kB = 128;  // elements per scale

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8;

// ===========================================================================
// Quantisation
// ===========================================================================

// |x| as ordered bits, 0 for a value that is not finite (it has no part in the scale).
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

// The e8m0 byte (e + 127) of a block whose largest |x| has these bits: with |x| =
// 1.f * 2^(E-127), 448 = 1.75 * 2^8 gives e = E - 135, one more above 1.75.
// Blocks below 2^-119 stay at 2^-127, a block of zeros is at 1.
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  const int b = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax == 0 ? 127 : (b > 0 ? b : 0);
}

// 2^-e, e in [-127, 120]: always a normal number, so the product with it is exact
// wherever e4m3 keeps anything of it.
__device__ __forceinline__ float inv_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// Four scaled values to four e4m3 bytes; a value that is not finite becomes NaN.
__device__ __forceinline__ float q_in(float x, float inv) {
  return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u ? x * inv : __builtin_nanf("");
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
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

struct QuantArgs {
  int64_t rows, cols;
  const void* x;
  int64_t ldx;
  int vec;      // rows start on 16 bytes
  int group;    // rows per scale: 1 or 128
  uint8_t* q;   // blocks along the columns (may be null)
  int64_t ldq;
  uint8_t* s;
  int64_t lds;
  uint8_t* qt;  // the transpose, blocks along the rows (may be null)
  int64_t ldqt;
  uint8_t* st;
  int64_t ldst;
};

// x[row][c0 .. c0+7] as floats, zero past the last column
template <typename T>
__device__ __forceinline__ void load8(const QuantArgs& a, int64_t row, int64_t c0, float v[8]) {
  const T* p = reinterpret_cast<const T*>(a.x) + row * a.ldx + c0;
  if (a.vec && c0 + 8 <= a.cols) {
    if constexpr (sizeof(T) == 2) {
      const u32x4 u = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_lo(u[i]);
        v[2 * i + 1] = bf16_hi(u[i]);
      }
    } else {
      const f32x4 u0 = reinterpret_cast<const f32x4*>(p)[0], u1 = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = u0[i];
        v[4 + i] = u1[i];
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float f = 0.f;
    if (c0 + i < a.cols) {
      if constexpr (sizeof(T) == 2) f = bf16_to_f32(p[i]);
      else f = p[i];
    }
    v[i] = f;
  }
}

// One row's block of 128 per 16 lanes, 8 elements a lane: one read, one write.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a, uint32_t blocks, uint32_t kb) {
  const uint32_t id = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (id >= blocks) return;  // whole groups of 16 lanes leave together
  const uint32_t row = id / kb, b = id - row * kb;
  const int l = threadIdx.x & 15;
  const int64_t c0 = (int64_t)b * kB + l * 8;
  float v[8];
  load8<T>(a, row, c0, v);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, finite_abs_bits(v[i]));
  const int byte = scale_byte(max16(m));
  const float inv = inv_scale(byte);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = q_in(v[i], inv);
  *reinterpret_cast<u32x2*>(a.q + (int64_t)row * a.ldq + c0) =
      u32x2{pack_e4m3x4(v[0], v[1], v[2], v[3]), pack_e4m3x4(v[4], v[5], v[6], v[7])};
  if (l == 0) a.s[(int64_t)row * a.lds + b] = (uint8_t)byte;
}

// A 128 x 128 tile per workgroup: read once, written along the rows and, through
// LDS, along the columns. Lane group g = tid / 16 holds rows 8g .. 8g+7, lane
// l = tid % 16 columns 8l .. 8l+7, so a thread has the 8 bytes of a column that
// lie together in the transpose.
template <typename T>
__global__ __launch_bounds__(256) void quantize_tile_kernel(QuantArgs a) {
  __shared__ uint32_t colmax[16][kB];
  __shared__ uint8_t colbyte[kB];
  __shared__ __attribute__((aligned(16))) u32x2 tile[kB * 16];  // [column][8-row slot ^ (column / 8)]
  const int tid = threadIdx.x, l = tid & 15, g = tid >> 4;
  const int64_t r0 = (int64_t)blockIdx.y * kB, c0 = (int64_t)blockIdx.x * kB;
  const int64_t cl = c0 + l * 8;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + g * 8 + i;
    if (r < a.rows) {
      load8<T>(a, r, cl, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  uint32_t rm[8], cm[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    rm[i] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t u = finite_abs_bits(v[i][j]);
      rm[i] = max(rm[i], u);
      cm[j] = max(cm[j], u);
    }
  }
  if (a.group != 1 || a.qt) {
#pragma unroll
    for (int j = 0; j < 8; ++j) colmax[g][l * 8 + j] = cm[j];
    __syncthreads();
    if (tid < kB) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) m = max(m, colmax[i][tid]);
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
    for (int i = 0; i < 8; ++i) {
      const int64_t r = r0 + g * 8 + i;
      const int byte = a.group != 1 ? one : scale_byte(max16(rm[i]));
      if (r >= a.rows) continue;
      const float inv = inv_scale(byte);
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = q_in(v[i][j], inv);
      *reinterpret_cast<u32x2*>(a.q + r * a.ldq + cl) =
          u32x2{pack_e4m3x4(w[0], w[1], w[2], w[3]), pack_e4m3x4(w[4], w[5], w[6], w[7])};
      if (l == 0 && a.group == 1) a.s[r * a.lds + blockIdx.x] = (uint8_t)byte;
    }
    if (a.group != 1 && tid == 0) a.s[(int64_t)blockIdx.y * a.lds + blockIdx.x] = (uint8_t)one;
  }
  if (!a.qt) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = l * 8 + j;
    const float inv = inv_scale(a.group != 1 ? one : colbyte[c]);
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = q_in(v[i][j], inv);
    tile[c * 16 + (g ^ l)] = u32x2{pack_e4m3x4(w[0], w[1], w[2], w[3]), pack_e4m3x4(w[4], w[5], w[6], w[7])};
  }
  __syncthreads();
  // 8 lanes write a column's 128 bytes, 16 a lane
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int c = it * 32 + (tid >> 3), h = tid & 7;
    if (c0 + c >= a.cols) continue;
    const u32x2 lo = tile[c * 16 + ((2 * h) ^ (c >> 3))], hi = tile[c * 16 + ((2 * h + 1) ^ (c >> 3))];
    *reinterpret_cast<u32x4*>(a.qt + (c0 + c) * a.ldqt + r0 + h * 16) = u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
  if (a.group == 1) {
    if (tid < kB && c0 + tid < a.cols) a.st[(c0 + tid) * a.ldst + blockIdx.y] = colbyte[tid];
  } else if (tid == 0) {
    a.st[(int64_t)blockIdx.x * a.ldst + blockIdx.y] = (uint8_t)one;
  }
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
//     columns; rows leave through LDS in whole 16-byte pieces.

struct GemmF8Args {
  int M, N, K, Kp;
  const uint8_t* A;
  int64_t lda;
  const uint8_t* sa;
  int64_t ldsa;
  int sha;  // log2 of the rows per scale: 0 or 7
  int dwa;  // scale rows are whole, aligned dwords
  const uint8_t* B;
  int64_t ldb;
  const uint8_t* sb;
  int64_t ldsb;
  int shb, dwb;
  void* C;
  int64_t ldc;
  float* ws;     // split partials [splits][M][ldw], or null
  int64_t ldw;
  int tiles;     // output tiles
  int kb_chunk;  // blocks per split (a multiple of 4 when there is more than one)
};

// Scale bytes 4q .. 4q+3 of one row (nkb of them there): one dword where rows
// start on 4 bytes and are padded to whole dwords, else byte by byte.
__device__ __forceinline__ uint32_t scales4(const uint8_t* p, int q, int nkb, int dw) {
  if (dw) return reinterpret_cast<const uint32_t*>(p)[q];
  uint32_t v = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    if (4 * q + b < nkb) v |= (uint32_t)p[4 * q + b] << (8 * b);
  return v;
}

// 16 e4m3 bytes times a power of two (given as the float it is) to two fragments
// of 8 bf16. Exact: 4 significant bits in 8, and bf16 has the range of the scales.
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

// One MFMA, then its share of the R fragment reads of the next step.
template <int M, int NM, int R>
__device__ __forceinline__ void sched_f8() {
  if constexpr (M < NM) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    constexpr int lo = M * R / NM, hi = (M + 1) * R / NM;
    if constexpr (hi > lo) __builtin_amdgcn_sched_group_barrier(0x100, hi - lo, 0);
    sched_f8<M + 1, NM, R>();
  }
}

template <int BM, int BN, int WTM, int WTN, typename OutT>
__global__ __launch_bounds__((BM / WTM) * (BN / WTN) * 64, (BM * BN >= 65536) ? 1 : 2) void gemm_f8_kernel(
    GemmF8Args g) {
  constexpr int WNW = BN / WTN, NWV = (BM / WTM) * WNW;
  constexpr int FM = WTM / 32, FN = WTN / 32;
  constexpr int STAGE = (BM + BN) * kB;
  constexpr int IA = BM / 8 / NWV, IB = BN / 8 / NWV;  // DMA instructions (8 rows each) per wave and stage
  static_assert(IA * 8 * NWV == BM && IB * 8 * NWV == BN, "a stage splits into whole DMA instructions");
  constexpr bool kWide = sizeof(OutT) == 4;            // widened to bf16 for fp32 sums
  constexpr int NS = kWide ? 4 : 2;                    // fragment steps of a stage: 16 or 32 bytes of k a lane
  constexpr int CH = kWide ? 1 : 2;                    // 16-byte chunks of a fragment
  __shared__ __attribute__((aligned(16))) uint8_t st0[STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t st1[STAGE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WNW, wn = wave % WNW;

  // each XCD takes a contiguous run of tiles, in groups of 8 tile rows
  int bid = blockIdx.x;
  {
    const int nwg = gridDim.x, per = nwg / 8;
    if (bid < per * 8) bid = (bid % 8) * per + bid / 8;
  }
  const int tiles_n = (g.N + BN - 1) / BN;
  const int tiles_m = (g.M + BM - 1) / BM;
  const int split = bid / g.tiles;
  const int tile = bid - split * g.tiles;
  constexpr int GM = 8;
  const int in_group = GM * tiles_n;
  const int first_m = (tile / in_group) * GM;
  const int gsize = min(tiles_m - first_m, GM);
  const int tm = first_m + (tile % in_group) % gsize;
  const int tn = (tile % in_group) / gsize;
  const int m0 = tm * BM, n0 = tn * BN;
  const int kb0 = split * g.kb_chunk;
  const int nkb = min(g.Kp / kB, kb0 + g.kb_chunk) - kb0;  // blocks of this split

  // Descriptors start at the tile's first row (64-bit base), so 32-bit offsets
  // reach any matrix; rows past the last one read as zero.
  const int ra_rows = min(g.M - m0, BM), rb_rows = min(g.N - n0, BN);
  const uint8_t* pa = g.A + (int64_t)m0 * g.lda;
  const uint8_t* pb = g.B + (int64_t)n0 * g.ldb;
  const uint32_t ba = (uint32_t)((int64_t)(ra_rows - 1) * g.lda + g.Kp);
  const uint32_t bb = (uint32_t)((int64_t)(rb_rows - 1) * g.ldb + g.Kp);
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
  auto issue = [&](uint8_t* sb, int kt) __attribute__((always_inline)) {
    // behind the last stage an empty descriptor reads nothing: a branch here would let
    // the compiler move the MFMAs before it to the ones behind it
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(pa, kt < nkb ? ba : 0), rb = make_rsrc(pb, kt < nkb ? bb : 0);
    const uint32_t soff = (uint32_t)(kb0 + kt) * kB;
#pragma unroll
    for (int i = 0; i < IA; ++i) dma16(ra, sb + (i * NWV + wave) * 1024, va[i], soff);
#pragma unroll
    for (int i = 0; i < IB; ++i) dma16(rb, sb + BM * kB + (i * NWV + wave) * 1024, vb[i], soff);
  };

  // scale rows of this lane's fragments (byte offsets from the tile's first), four blocks to a dword
  const uint8_t* psa = g.sa + (int64_t)(m0 >> g.sha) * g.ldsa + kb0;
  const uint8_t* psb = g.sb + (int64_t)(n0 >> g.shb) * g.ldsb + kb0;
  uint32_t osa[FM], osb[FN];
  const int frow = lane & 31;
#pragma unroll
  for (int i = 0; i < FM; ++i)
    osa[i] = (uint32_t)((min(wm * WTM + i * 32 + frow, ra_rows - 1) >> g.sha) * g.ldsa);
#pragma unroll
  for (int j = 0; j < FN; ++j)
    osb[j] = (uint32_t)((min(wn * WTN + j * 32 + frow, rb_rows - 1) >> g.shb) * g.ldsb);
  uint32_t sca[FM], scb[FN], nca[FM], ncb[FN];
  auto load_scales = [&](int q) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FM; ++i) nca[i] = scales4(psa + osa[i], q, nkb, g.dwa);
#pragma unroll
    for (int j = 0; j < FN; ++j) ncb[j] = scales4(psb + osb[j], q, nkb, g.dwb);
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
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  auto compute = [&](int in, auto pos) __attribute__((always_inline)) {
    constexpr int P = decltype(pos)::value;  // the block's byte in the scale dwords
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
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma32(b[j][h], a[h], acc[i][j]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[in][j], fa[in][i], acc[i][j], 0, 0, P,
                                                                     (int)scb[j], P, (int)sca[i]);
    }
  };

  // Stage kt: every step reads the next one's fragments while its MFMAs run. The
  // last step's fragments are in registers when the workgroup meets, so the stage's
  // buffer is free for stage kt + 2 and the first fragments of kt + 1 (whose DMA has
  // had a whole stage to land) are read under the last step's MFMAs.
  auto stage = [&](int kt, auto pos) __attribute__((always_inline)) {
    uint8_t* cur = decltype(pos)::value % 2 == 0 ? st0 : st1;
    uint8_t* nxt = decltype(pos)::value % 2 == 0 ? st1 : st0;
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      if (t + 1 < NS) {
        read(cur, t + 1, (t + 1) & 1);
      } else {
        wait_vm<0>();
        __syncthreads();
        issue(cur, kt + 2);
        read(nxt, 0, 0);  // (behind the last stage: not used)
      }
      compute(t & 1, pos);
      if constexpr (!kWide) sched_f8<0, FM * FN, (FM + FN) * CH>();
    }
  };
  using P0 = std::integral_constant<int, 0>;
  using P1 = std::integral_constant<int, 1>;
  using P2 = std::integral_constant<int, 2>;
  using P3 = std::integral_constant<int, 3>;
  auto next_scales = [&](int kt) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FM; ++i) sca[i] = nca[i];
#pragma unroll
    for (int j = 0; j < FN; ++j) scb[j] = ncb[j];
    load_scales(min((kt >> 2) + 1, (nkb - 1) >> 2));
  };
  int kt = 0;
  if (nkb > 0) {
    load_scales(0);
    issue(st0, 0);
    issue(st1, 1);
    wait_vm<IA + IB>();
    __syncthreads();
    read(st0, 0, 0);
    for (; kt + 4 <= nkb; kt += 4) {
      next_scales(kt);
      stage(kt, P0{});
      stage(kt + 1, P1{});
      stage(kt + 2, P2{});
      stage(kt + 3, P3{});
    }
    if (kt < nkb) {
      next_scales(kt);
      stage(kt, P0{});
      if (kt + 1 < nkb) {
        stage(kt + 1, P1{});
        if (kt + 2 < nkb) stage(kt + 2, P2{});
      }
    }
  }

  const int g4 = (lane >> 5) * 4;
  if (g.ws) {
    float* W = g.ws + (int64_t)split * g.M * g.ldw;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = m0 + wm * WTM + i * 32 + frow;
      if (m >= g.M) continue;
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + wn * WTN + j * 32 + q * 8 + g4;
          if (n < g.N)
            *reinterpret_cast<f32x4*>(W + (int64_t)m * g.ldw + n) =
                f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        }
    }
    return;
  }
  // Each wave passes 32 rows at a time through its own LDS slab and stores rows
  // in 16-byte pieces (a lane's own results are pieces of 32 different rows).
  __syncthreads();
  constexpr int PITCH = WTN * (int)sizeof(OutT), CPR = PITCH / 16, EPC = 16 / (int)sizeof(OutT), RPI = 64 / CPR;
  static_assert(NWV * 32 * PITCH <= STAGE, "the slabs fit the first stage");
  static_assert(CPR <= 64, "a row is one instruction's pieces at most");
  uint8_t* wl = st0 + wave * 32 * PITCH;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int cb = (j * 32 + q * 8 + g4) * (int)sizeof(OutT);
        uint8_t* at = wl + frow * PITCH + (((cb >> 4) ^ (frow & (CPR - 1))) << 4) + (cb & 15);
        const float x0 = acc[i][j][4 * q], x1 = acc[i][j][4 * q + 1], x2 = acc[i][j][4 * q + 2],
                    x3 = acc[i][j][4 * q + 3];
        if constexpr (sizeof(OutT) == 2) *reinterpret_cast<u32x2*>(at) = u32x2{pack_bf16x2(x0, x1), pack_bf16x2(x2, x3)};
        else *reinterpret_cast<f32x4*>(at) = f32x4{x0, x1, x2, x3};
      }
#pragma unroll
    for (int it = 0; it < 32 / RPI; ++it) {
      const int r = it * RPI + lane / CPR, ch = lane % CPR;
      const u32x4 val = *reinterpret_cast<const u32x4*>(wl + r * PITCH + ((ch ^ (r & (CPR - 1))) << 4));
      const int m = m0 + wm * WTM + i * 32 + r;
      const int n = n0 + wn * WTN + ch * EPC;
      if (m >= g.M || n >= g.N) continue;
      OutT* dst = reinterpret_cast<OutT*>(g.C) + (int64_t)m * g.ldc + n;
      if (n + EPC <= g.N) {
        __builtin_nontemporal_store(val, reinterpret_cast<u32x4*>(dst));
      } else {
#pragma unroll
        for (int k = 0; k < EPC; ++k) {
          if (n + k >= g.N) break;
          if constexpr (sizeof(OutT) == 2) dst[k] = (OutT)(val[k >> 1] >> (16 * (k & 1)));
          else dst[k] = __uint_as_float(val[k]);
        }
      }
    }
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

struct F8Plan {
  bool huge;
  int tiles, splits, kb_chunk;
};

F8Plan f8_plan(int M, int N, int K) {
  const int64_t kb = ((int64_t)K + kB - 1) / kB;
  auto tiles = [&](int t) { return (((int64_t)M + t - 1) / t) * (((int64_t)N + t - 1) / t); };
  F8Plan p;
  p.huge = tiles(256) >= 256;
  const int64_t t = tiles(p.huge ? 256 : 128);
  int64_t s = 1;
  if (!p.huge && t < 256) s = std::max<int64_t>(1, std::min<int64_t>(512 / t, kb / 4));
  const int64_t chunk = s > 1 ? ((kb + s - 1) / s + 3) / 4 * 4 : std::max<int64_t>(kb, 1);
  p.splits = (int)std::max<int64_t>(1, (kb + chunk - 1) / chunk);
  p.kb_chunk = (int)chunk;
  p.tiles = t > INT32_MAX ? -1 : (int)t;
  return p;
}

int64_t f8_ldw(int N) { return ((int64_t)N + 3) / 4 * 4; }

template <typename OutT>
void launch_f8(hipStream_t st, const F8Plan& p, const GemmF8Args& g) {
  const dim3 grid((unsigned)(p.tiles * p.splits));
  if (p.huge)
    hipLaunchKernelGGL((gemm_f8_kernel<256, 256, 128, 128, OutT>), grid, dim3(256), 0, st, g);
  else
    hipLaunchKernelGGL((gemm_f8_kernel<128, 128, 64, 64, OutT>), grid, dim3(256), 0, st, g);
  if (p.splits > 1)
    hipLaunchKernelGGL((f8_reduce_kernel<OutT>),
                       dim3((unsigned)((g.N + 255) / 256), (unsigned)std::min<int64_t>(((int64_t)g.M + 3) / 4, 65535)),
                       dim3(256), 0, st, g, p.splits);
}

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

extern "C" int nl_quantize_fp8(void* stream, int64_t rows, int64_t cols, const void* x, int x_dtype, int64_t ldx,
                               int group, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds, uint8_t* qt,
                               int64_t ldqt, uint8_t* scale_t, int64_t ldst) {
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > INT32_MAX)
    return nl_set_error(NL_EINVAL, "quantize_fp8: need 0 <= rows, cols < 2^31");
  if (x_dtype != NL_DTYPE_F32 && x_dtype != NL_DTYPE_BF16)
    return nl_set_error(NL_EINVAL, "quantize_fp8: x is fp32 or bf16");
  if (!q && !qt) return nl_set_error(NL_EINVAL, "quantize_fp8: no output");
  if (q)
    if (int rc = check_operand("quantize_fp8", rows, cols, q, ldq, scale, lds, group)) return rc;
  if (qt)
    if (int rc = check_operand("quantize_fp8 (transpose)", cols, rows, qt, ldqt, scale_t, ldst, group)) return rc;
  if (rows == 0 || cols == 0) return NL_OK;
  const int esz = x_dtype == NL_DTYPE_BF16 ? 2 : 4;
  if (!x) return nl_set_error(NL_EINVAL, "quantize_fp8: null x");
  if (rows > 1 && ldx < cols) return nl_set_error(NL_EINVAL, "quantize_fp8: ldx < cols");
  if ((uintptr_t)x % esz) return nl_set_error(NL_EALIGN, "quantize_fp8: x is not aligned to its type");
  const int64_t rb = (rows + kB - 1) / kB, cb = (cols + kB - 1) / kB;
  QuantArgs a{rows, cols, x, ldx, (((uintptr_t)x & 15) == 0 && (rows == 1 || ldx * esz % 16 == 0)) ? 1 : 0, group,
              q, ldq, scale, lds, qt, ldqt, scale_t, ldst};
  hipStream_t st = (hipStream_t)stream;
  if (!qt && group == 1) {
    const int64_t blocks = rows * cb;
    if (blocks > INT32_MAX) return nl_set_error(NL_EUNSUPPORTED, "quantize_fp8: more than 2^31 blocks");
    const dim3 grid((unsigned)((blocks + 15) / 16));
    if (esz == 2)
      hipLaunchKernelGGL((quantize_rows_kernel<uint16_t>), grid, dim3(256), 0, st, a, (uint32_t)blocks, (uint32_t)cb);
    else
      hipLaunchKernelGGL((quantize_rows_kernel<float>), grid, dim3(256), 0, st, a, (uint32_t)blocks, (uint32_t)cb);
    return nl_check_launch("nl_quantize_fp8");
  }
  if (rb > 65535) return nl_set_error(NL_EUNSUPPORTED, "quantize_fp8: more than 65535 blocks of rows");
  const dim3 grid((unsigned)cb, (unsigned)rb);
  if (esz == 2)
    hipLaunchKernelGGL((quantize_tile_kernel<uint16_t>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((quantize_tile_kernel<float>), grid, dim3(256), 0, st, a);
  return nl_check_launch("nl_quantize_fp8");
}

extern "C" size_t nl_gemm_fp8_ws_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const F8Plan p = f8_plan(M, N, K);
  return p.splits > 1 ? (size_t)p.splits * M * f8_ldw(N) * sizeof(float) : 0;
}

extern "C" int nl_gemm_fp8(void* stream, int M, int N, int K, const uint8_t* A, int64_t lda, const uint8_t* scale_a,
                           int64_t ldsa, int group_a, const uint8_t* B, int64_t ldb, const uint8_t* scale_b,
                           int64_t ldsb, int group_b, void* C, int c_dtype, int64_t ldc, void* ws, size_t ws_bytes) {
  if (M < 0 || N < 0 || K < 0) return nl_set_error(NL_EINVAL, "gemm_fp8: need M, N, K >= 0");
  if (c_dtype != NL_DTYPE_F32 && c_dtype != NL_DTYPE_BF16)
    return nl_set_error(NL_EINVAL, "gemm_fp8: C is fp32 or bf16");
  if (int rc = check_operand("gemm_fp8 A", M, K, A, lda, scale_a, ldsa, group_a)) return rc;
  if (int rc = check_operand("gemm_fp8 B", N, K, B, ldb, scale_b, ldsb, group_b)) return rc;
  if (M == 0 || N == 0) return NL_OK;
  if (!C) return nl_set_error(NL_EINVAL, "gemm_fp8: null C");
  if (ldc < N) return nl_set_error(NL_EINVAL, "gemm_fp8: ldc < N");
  if (((uintptr_t)C & 15) || ldc % 8) return nl_set_error(NL_EALIGN, "gemm_fp8: C needs 16-byte aligned rows");
  const int64_t Kp = ((int64_t)K + kB - 1) / kB * kB;
  // 256 rows of a tile are addressed with 31-bit offsets
  if (lda > INT32_MAX / 256 || ldb > INT32_MAX / 256 || Kp > INT32_MAX / 256)
    return nl_set_error(NL_EUNSUPPORTED, "gemm_fp8: rows of 8 MiB and more");
  F8Plan p = f8_plan(M, N, K);
  if (p.tiles < 0 || (int64_t)p.tiles * p.splits > INT32_MAX) return nl_set_error(NL_EUNSUPPORTED, "gemm_fp8: too many tiles");
  auto dwords = [](const void* s, int64_t ld) { return (int)(ld % 4 == 0 && ((uintptr_t)s & 3) == 0); };
  GemmF8Args g{M, N, K, (int)Kp,
               A, lda, scale_a, ldsa, group_a == kB ? 7 : 0, dwords(scale_a, ldsa),
               B, ldb, scale_b, ldsb, group_b == kB ? 7 : 0, dwords(scale_b, ldsb),
               C, ldc, nullptr, f8_ldw(N), p.tiles, p.kb_chunk};
  if (p.splits > 1) {
    if (ws && ws_bytes >= nl_gemm_fp8_ws_bytes(M, N, K)) {
      if ((uintptr_t)ws & 15) return nl_set_error(NL_EALIGN, "gemm_fp8: workspace not 16-byte aligned");
      g.ws = (float*)ws;
    } else {
      p.splits = 1;
      g.kb_chunk = (int)(Kp / kB);
    }
  }
  if (c_dtype == NL_DTYPE_F32) launch_f8<float>((hipStream_t)stream, p, g);
  else launch_f8<uint16_t>((hipStream_t)stream, p, g);
  return nl_check_launch("nl_gemm_fp8");
}
