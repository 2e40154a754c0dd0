// distill.hip — distillation from a teacher's top logits, for gfx950.
//
//   top:   the k largest of x[m, :], ties to the lowest index, and
//          lse[m] = log sum_v exp(x[m, v] / T)
//   loss:  p_j = exp(v_j / T - lse_t)  (or the softmax of the row's v_j / T)
//          loss[m] = T^2 sum_j p_j (log p_j - log q[id_j]),  q = softmax(z[m] / T)
//          dz[m, v] = scale T (S q_v - sum_{j: id_j = v} p_j),  S = sum_j p_j
//
// Both are bound by HBM: a row of logits is read once into registers by one
// workgroup (as the cross-entropy does), and every pass over it runs from there.
// Rows that no workgroup's registers hold (beyond 106503 logits) are read twice.
// Measured at 16384 x 50257, k = 64: the loss with its gradient 646 us (5.1 TB/s; a copy
// reaches 4.7), the loss alone 327 us (5.0 TB/s), the top logits 410 us (4.0 TB/s). At 4096 x
// 106503, in registers, 380, 173 and 297 us; at 4096 x 128256, read twice, 478, 183 and 432.
// Every difference from a row's largest value is formed before a logarithm is added to it:
// logits may be masks of any finite size, and a row may stand far from zero.
#include "common.h"

namespace nl {
namespace {

constexpr int kMaxK = NL_TOP_MAX_K;

// 2^x for x of any size with the error of a small argument: the integer part goes
// into the exponent exactly. 0 at -inf, NaN at NaN.
__device__ __forceinline__ float exp2_split(double x) {
  if (x < -300.0) return 0.f;
  if (x > 300.0) return INFINITY;
  const double n = rint(x);
  return ldexpf(fast_exp2((float)(x - n)), (int)n);
}

// A row of V bf16 values held by a workgroup of NT threads: 8-element vectors in
// NVEC registers sets per thread (0: left in memory and read again), and at most
// one loose element (before the first or behind the last 16-byte boundary).
template <int NT, int NVEC>
struct Row {
  const uint16_t* p;
  const u32x4* body;
  int V, head, nbody, eidx;
  u32x4 v[NVEC ? NVEC : 1];
  float top[NVEC ? NVEC : 1];  // largest of each vector (NaN apart), where row_sums is asked for it
  float xe;  // the loose element

  __device__ __forceinline__ void load(const uint16_t* row, int n, int tid) {
    p = row;
    V = n;
    const int mis = (int)(((uintptr_t)row & 15) >> 1);
    head = min(mis ? 8 - mis : 0, V);
    nbody = (V - head) >> 3;
    const int tail = (V - head) & 7;
    body = reinterpret_cast<const u32x4*>(row + head);
#pragma unroll
    for (int j = 0; j < NVEC; ++j)
      if (j * NT + tid < nbody) v[j] = __builtin_nontemporal_load(body + j * NT + tid);
    eidx = -1;
    if (tid < head) eidx = tid;
    else if (tid >= 8 && tid < 8 + tail) eidx = head + nbody * 8 + (tid - 8);
    xe = eidx >= 0 ? bf16_to_f32(row[eidx]) : 0.f;
  }
  // keeps the row packed between passes (unpacked floats would take twice the registers)
  __device__ __forceinline__ void fence() {
#pragma unroll
    for (int j = 0; j < NVEC; ++j) asm volatile("" : "+v"(v[j]));
  }
  // f(vector, index of its first element / 8 in the body, j) for this thread's vectors
  template <class F>
  __device__ __forceinline__ void vectors(int tid, F f) {
    if constexpr (NVEC > 0) {
#pragma unroll
      for (int j = 0; j < NVEC; ++j)
        if (j * NT + tid < nbody) f(v[j], j * NT + tid, j);
    } else {
      for (int i = tid; i < nbody; i += NT) f(body[i], i, 0);
    }
  }
};

template <int NT>
struct RowSums {
  float m[NT / kWave], s[NT / kWave];
};

// (X, S) over the workgroup's row: X = max x and S = sum 2^((x - X) c). A NaN makes S NaN; an infinity without one makes both infinite.
__device__ __forceinline__ float finite_or_0(float m) { return fabsf(m) == INFINITY ? 0.f : m; }
__device__ __forceinline__ void combine(float& m, float& s, float m2, float s2, float c) {
  const float mn = fmaxf(m, m2);
  const float at = finite_or_0(mn);
  s = s * fast_exp2((m - at) * c) + s2 * fast_exp2((m2 - at) * c);
  m = mn;
}

// Sums over a row take 2^(x c - off) with off = m c rounded, one fma an element, and multiply by
// 2^(off - m c) at the end. That rounding is at most 2^-24 |m| c, so 1/16 up to here; beyond it
// (masks of a large finite value) the factor would soon leave fp32, and (x - m) c is formed instead.
__device__ __forceinline__ bool is_far(float m, float c) { return !(fabsf(m) * c <= 1048576.f); }

__device__ __forceinline__ float max8(const u32x4& v) {
  float m = fmaxf(bf16_lo(v[0]), bf16_hi(v[0]));
#pragma unroll
  for (int q = 1; q < 4; ++q) m = fmaxf(m, fmaxf(bf16_lo(v[q]), bf16_hi(v[q])));
  return m;
}

// per_wave(thread's max) runs on every wave ahead of the workgroup's barrier.
template <bool kTops = false, int NT, int NVEC, class F>
__device__ __forceinline__ void row_sums(Row<NT, NVEC>& r, float c, int tid, RowSums<NT>& sm, float& X, float& S,
                                         F per_wave) {
  float m = r.eidx >= 0 ? r.xe : -INFINITY;
  float s;
  if constexpr (NVEC > 0) {
    r.vectors(tid, [&](const u32x4& v, int, int j) {
      const float t = max8(v);
      if constexpr (kTops) r.top[j] = t;
      m = fmaxf(m, t);
    });
    r.fence();
    auto sum = [&](auto f) __attribute__((always_inline)) {
      s = r.eidx >= 0 ? fast_exp2(f(r.xe)) : 0.f;
      r.vectors(tid, [&](const u32x4& v, int, int) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          s += fast_exp2(f(bf16_lo(v[q])));
          s += fast_exp2(f(bf16_hi(v[q])));
        }
      });
    };
    const float at = finite_or_0(m);
    if (!is_far(at, c)) {
      const float off = at * c;
      sum([&](float x) { return __builtin_fmaf(x, c, -off); });
      s *= fast_exp2(__builtin_fmaf(-at, c, off));
    } else {
      sum([&](float x) { return (x - at) * c; });
    }
    r.fence();
  } else {
    // one read: the running maximum moves once per vector at most
    float at = finite_or_0(m);
    s = r.eidx >= 0 ? fast_exp2((r.xe - at) * c) : 0.f;
    r.vectors(tid, [&](const u32x4& v, int, int) {
      const float mv = max8(v);
      if (mv > m) {
        const float to = finite_or_0(mv);
        s *= s == 0.f ? 1.f : fast_exp2((at - to) * c);  // (a sum of 0 has no reference yet)
        m = mv;
        at = to;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        s += fast_exp2((bf16_lo(v[q]) - at) * c);
        s += fast_exp2((bf16_hi(v[q]) - at) * c);
      }
    });
  }
  per_wave(m);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o, kWave);
    const float s2 = __shfl_xor(s, o, kWave);
    combine(m, s, m2, s2, c);
  }
  if constexpr (NT > kWave) {
    if ((tid & (kWave - 1)) == 0) {
      sm.m[tid / kWave] = m;
      sm.s[tid / kWave] = s;
    }
    __syncthreads();
    m = sm.m[0];
    s = sm.s[0];
#pragma unroll
    for (int w = 1; w < NT / kWave; ++w) combine(m, s, sm.m[w], sm.s[w], c);
  }
  X = m;
  S = s;
}

// ===========================================================================
// The k largest
// ===========================================================================
//
// Each wave finds the j-th largest of its lanes' maxima, j = ceil(k / waves): at least
// j of its elements reach that, so at least k of the row's reach the least of the
// waves' bounds, and with elements in no particular order hardly twice as many do.
// (Where j is a large part of the 64 lanes, and a row is short, the waves count over
// all their elements instead.) Those go to LDS as (key, index), a list for each wave,
// and their rank among each other is their place. A row with more of them than fit
// (ties, mostly), or with a NaN, goes over the row in memory again.
// At 16384 x 50257: 341 us for k = 1, 410 for 64, 566 for 256, of which the sums of the
// row take 327. (Before: every candidate ranked against all others, and each vector looked
// through where it was found: 397, 482 and 1112 us.)

// bf16 bits as an ordered 16-bit number: -0 as 0, every NaN above infinity
__device__ __forceinline__ uint32_t order16(uint32_t h) {
  if ((h & 0x7fff) > 0x7f80) return 0xffffu;
  if (h == 0x8000) h = 0;
  return (h & 0x8000) ? (~h & 0xffff) : (h | 0x8000);
}
// the number that has this order (-inf below all of them)
__device__ __forceinline__ float from_order16(uint32_t o) {
  return o <= 0x7f ? -INFINITY : bf16_to_f32((uint16_t)(o & 0x8000 ? o & 0x7fff : ~o & 0xffff));
}

// larger key first, then the lower index; the low 16 bits carry the value
__device__ __forceinline__ unsigned long long entry(uint32_t h, int i) {
  return ((unsigned long long)order16(h) << 48) | ((unsigned long long)(uint32_t)(~i) << 16) | h;
}

template <int NT>
__device__ __forceinline__ int block_count(int n, int tid, int* sm) {
  n = (int)wave_sum((float)n);  // counts stay below 2^24 (V < 2^24)
  if constexpr (NT > kWave) {
    __syncthreads();
    if ((tid & (kWave - 1)) == 0) sm[tid / kWave] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < NT / kWave; ++w) n += sm[w];
  }
  return n;
}

// The k largest of the row in memory into cand, exactly k of them. `key`: an order
// that at least k elements reach.
template <int NT>
__device__ __noinline__ void select_in_memory(const uint16_t* row, int V, int k, uint32_t key, int tid, int* cnt,
                                              int* count, unsigned long long* cand) {
  Row<NT, 0> r;
  r.load(row, V, tid);
  auto above = [&](uint32_t t) {  // elements with a larger order than t
    int m = r.eidx >= 0 && order16(__float_as_uint(r.xe) >> 16) > t;
#pragma unroll 4
    for (int i = tid; i < r.nbody; i += NT) {
      const u32x4 v = r.body[i];
#pragma unroll
      for (int q = 0; q < 4; ++q) m += (order16(v[q] & 0xffffu) > t) + (order16(v[q] >> 16) > t);
    }
    return block_count<NT>(m, tid, cnt);
  };
  // the k-th largest key: the bound itself where ties are what there is too much of
  int more = above(key);
  if (more >= k) {
    key = 0;
#pragma unroll 1
    for (int b = 15; b >= 0; --b)
      if (above((key | (1u << b)) - 1) >= k) key |= 1u << b;
    more = above(key);
  }
  // its equals in the order of their indices: each thread counts a stretch of the row
  const int len = (V + NT - 1) / NT, i0 = min(tid * len, V), i1 = min(i0 + len, V);
  int eq = 0;
#pragma unroll 4
  for (int i = i0; i < i1; ++i) eq += order16(row[i]) == key;
  int before = eq;  // inclusive over the wave's lanes
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int up = __shfl_up(before, o, kWave);
    if ((tid & (kWave - 1)) >= o) before += up;
  }
  __syncthreads();
  if ((tid & (kWave - 1)) == kWave - 1) cnt[tid / kWave] = before;
  if (tid == 0) *count = 0;
  __syncthreads();
  before -= eq;
  for (int w = 0; w < tid / kWave; ++w) before += cnt[w];
  const int want = k - more;  // >= 1 of the equals
#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    const uint32_t h = row[i], o = order16(h);
    if (o > key) cand[want + atomicAdd(count, 1)] = entry(h, i);
    else if (o == key && before < want) cand[before++] = entry(h, i);
  }
  __syncthreads();
}

template <int NT, int NVEC>
__global__ __launch_bounds__(NT) void top_kernel(int V, const uint16_t* __restrict__ logits, int64_t ld, int k,
                                                 float c, double inv_t, uint16_t* __restrict__ values,
                                                 int32_t* __restrict__ ids, float* __restrict__ lse) {
  constexpr int NW = NT / kWave;
  constexpr int kCand = NW == 1 ? 512 : 1024;            // candidates that are ranked
  constexpr int CAP = NW == 1 ? kCand : 2 * kCand / NW;  // and that a wave's list holds
  __shared__ RowSums<NT> sums;
  __shared__ uint32_t bounds[NW];
  __shared__ __attribute__((aligned(16))) unsigned long long list[NW][CAP];
  __shared__ __attribute__((aligned(16))) u32x4 held[NW][kWave];  // vectors with a candidate, and where they stand
  __shared__ int held_at[NW][kWave];
  __shared__ __attribute__((aligned(16))) unsigned long long cand[kCand];
  __shared__ int count;
  __shared__ int cnt[NW];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const uint16_t* xrow = logits + row * ld;
  Row<NT, NVEC> r;
  r.load(xrow, V, tid);
  float X, S;
  row_sums<true>(r, c, tid, sums, X, S, [&](float m) __attribute__((always_inline)) {
    const int want = (k + NW - 1) / NW;
    uint32_t bound = 0;
    if (NVEC > 0 && NVEC * NT <= 512 && want > 16) {
#pragma unroll 1
      for (int b = 15; b >= 0; --b) {
        const float t = from_order16(bound | (1u << b));
        int n = __popcll(__ballot(r.eidx >= 0 && r.xe >= t));
        r.vectors(tid, [&](const u32x4& v, int, int) {
#pragma unroll
          for (int q = 0; q < 4; ++q) n += __popcll(__ballot(bf16_lo(v[q]) >= t)) + __popcll(__ballot(bf16_hi(v[q]) >= t));
        });
        // (a lane without the vector counts nothing: take the largest, lane 0 has every one)
        if (__builtin_amdgcn_readfirstlane(n) >= want) bound |= 1u << b;
      }
    } else {
      const uint32_t mine = order16(__float_as_uint(m) >> 16);
#pragma unroll
      for (int b = 15; b >= 0; --b)
        if (__popcll(__ballot(mine >= (bound | (1u << b)))) >= want) bound |= 1u << b;
    }
    if (lane == 0) bounds[wave] = bound;
  });
  if constexpr (NT == kWave) __syncthreads();
  uint32_t bound = bounds[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) bound = min(bound, bounds[w]);
  bound = __builtin_amdgcn_readfirstlane(bound);
  const float fb = from_order16(bound);
  int n = 0;  // of this wave's list
  auto offer = [&](bool has, uint32_t h, int i) __attribute__((always_inline)) {
    const bool in = has && __uint_as_float(h << 16) >= fb;
    const unsigned long long mask = __ballot(in);
    if (mask == 0) return;
    const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    if (in && at < CAP) list[wave][at] = entry(h, i);
    n += __popcll(mask);
  };
  if (S == S) {
    offer(r.eidx >= 0, __float_as_uint(r.xe) >> 16, r.eidx);
    // Vectors that hold a candidate are few: they are gathered, one a lane, and looked
    // through together.
    int waiting = 0;
    auto look = [&]() __attribute__((always_inline)) {
      const bool has = lane < waiting;
      u32x4 v = {0, 0, 0, 0};
      int i = 0;
      __builtin_amdgcn_wave_barrier();
      if (has) {
        v = held[wave][lane];
        i = held_at[wave][lane];
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        offer(has, v[q] & 0xffffu, i + 2 * q);
        offer(has, v[q] >> 16, i + 2 * q + 1);
      }
      waiting = 0;
    };
    auto hold = [&](bool has, const u32x4& v, int i) __attribute__((always_inline)) {
      const unsigned long long mask = __ballot(has);
      if (mask == 0) return;
      const int more = __popcll(mask);
      if (waiting + more > kWave) look();
      if (has) {
        const int at =
            waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        held[wave][at] = v;
        held_at[wave][at] = r.head + i * 8;
      }
      waiting += more;
    };
    if constexpr (NVEC > 0) {
#pragma unroll
      for (int j = 0; j < NVEC; ++j)
        hold(j * NT + tid < r.nbody && r.top[j] >= fb, r.v[j], j * NT + tid);
    } else {
      for (int i0 = wave * kWave; i0 < r.nbody; i0 += NT) {
        const int i = i0 + lane;
        u32x4 v = {0, 0, 0, 0};
        if (i < r.nbody) v = r.body[i];
        hold(i < r.nbody && max8(v) >= fb, v, i);
      }
    }
    look();
  } else {
    n = CAP + 1;
  }
  if (lane == 0) cnt[wave] = n;
  __syncthreads();
  int total = 0, before = 0, most = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int m = cnt[w];
    if (w < wave) before += m;
    total += m;
    most = max(most, m);
  }
  if (most <= CAP && total <= kCand) {
    // each wave sorts its list by counting; then a candidate's rank is its place there
    // and, by bisection, the number of larger ones in every other list
    for (int i = lane; i < n; i += kWave) {
      const unsigned long long me = list[wave][i];
      int at = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) at += list[wave][j] > me;
      if (NW > 1) {
        cand[before + at] = me;
      } else if (at < k) {
        values[row * k + at] = (uint16_t)me;
        ids[row * k + at] = (int32_t)~(uint32_t)(me >> 16);
      }
    }
    if constexpr (NW > 1) {
      __syncthreads();
      int half = 1;
      while (half * 2 <= most) half *= 2;
      for (int i = tid; i < total; i += NT) {
        const unsigned long long me = cand[i];
        int at[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) at[w] = 0;
        for (int step = half; step > 0; step >>= 1) {
          int off = 0;
#pragma unroll
          for (int w = 0; w < NW; ++w) {
            const int m = cnt[w], to = at[w] + step;
            if (to <= m && cand[off + to - 1] > me) at[w] = to;
            off += m;
          }
        }
        int rank = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) rank += at[w];
        if (rank < k) {
          values[row * k + rank] = (uint16_t)me;
          ids[row * k + rank] = (int32_t)~(uint32_t)(me >> 16);
        }
      }
    }
  } else {
    select_in_memory<NT>(xrow, V, k, S == S ? bound : 0, tid, cnt, &count, cand);
    for (int i = tid; i < k; i += NT) {
      const unsigned long long me = cand[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < k; ++j) rank += cand[j] > me;
      values[row * k + rank] = (uint16_t)me;
      ids[row * k + rank] = (int32_t)~(uint32_t)(me >> 16);
    }
  }
  // X / T in 64 bits: c's rounding would be as much as the logarithm where X / T is large
  if (tid == NT - 1) lse[row] = (float)((double)X * inv_t + log2((double)S) * 0.69314718055994530942);
}

// ===========================================================================
// The loss and its gradient
// ===========================================================================

struct DistillArgs {
  int V, k;
  const uint16_t* z;
  int64_t ld;
  const void* ids;
  int ids_64;
  const void* values;
  int values_f32;
  const float* lse;  // null: softmax over the row's entries
  double inv_t;      // 1 / T
  float c;           // the same in 32 bits: the temperature that the student's row is taken at
  float t2ln2;       // T^2 ln 2
  float grad;        // scale T
  float* loss;
  uint16_t* dz;      // may be z itself
  int64_t ldd;
  int same_phase;    // rows of dz start at the same offset from 16 bytes as those of z
};

template <int NT, int NVEC, bool kGrad>
__global__ __launch_bounds__(NT) void distill_kernel(DistillArgs a) {
  __shared__ RowSums<NT> sums;
  __shared__ int sid[kMaxK];     // -1: padding
  __shared__ float sp[kMaxK];    // p_j
  __shared__ float sz[kMaxK];    // z[id_j]
  __shared__ double slp[kMaxK];  // log2 p_j
  __shared__ float sS;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const uint16_t* zrow = a.z + row * a.ld;
  Row<NT, NVEC> r;
  r.load(zrow, a.V, tid);
  // The first wave takes the teacher's entries, up to 4 a lane. They count in 64
  // bits: the loss is a difference of logarithms that may nearly cancel. v / T - lse is
  // rounded once: of two rounded products, 1.4e30 each, the rest would be 1e14.
  if (tid < kWave) {
    double lp[kMaxK / kWave];
    bool bad = false;
    double mx = -INFINITY;
    constexpr double kLog2e64 = 1.4426950408889634074;
    const double sub = a.lse ? (double)a.lse[row] : 0.0;
#pragma unroll
    for (int e = 0; e < kMaxK / kWave; ++e) {
      const int j = e * kWave + lane;
      lp[e] = -INFINITY;
      if (e * kWave >= a.k || j >= a.k) continue;
      const int64_t at = row * a.k + j;
      const int64_t id = a.ids_64 ? reinterpret_cast<const int64_t*>(a.ids)[at]
                                  : (int64_t)reinterpret_cast<const int32_t*>(a.ids)[at];
      sid[j] = id < 0 ? -1 : (id < a.V ? (int)id : -2);
      float z = 0.f;
      if (id >= 0) {
        const float v = a.values_f32 ? reinterpret_cast<const float*>(a.values)[at]
                                     : bf16_to_f32(reinterpret_cast<const uint16_t*>(a.values)[at]);
        lp[e] = __builtin_fma((double)v, a.inv_t, -sub);
        if (id < a.V) z = bf16_to_f32(zrow[id]);
        else lp[e] = __builtin_nan("");
        bad |= lp[e] != lp[e];
        mx = fmax(mx, lp[e]);
      }
      sz[j] = z;
    }
    if (!a.lse) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor(mx, o, kWave));
      const double at = mx == -INFINITY ? 0.0 : mx;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < kMaxK / kWave; ++e)
        if (e * kWave < a.k) s += exp2_split((lp[e] - at) * kLog2e64);
      s = wave_sum(s);
      // (the largest comes off first: beside a value of 1e17 the logarithm would be lost)
      const double l = s == 0.f ? 0.0 : log2((double)s);
#pragma unroll
      for (int e = 0; e < kMaxK / kWave; ++e) lp[e] = (lp[e] - at) * kLog2e64 - l;
    } else {
#pragma unroll
      for (int e = 0; e < kMaxK / kWave; ++e) lp[e] *= kLog2e64;
    }
    float S = 0.f;
#pragma unroll
    for (int e = 0; e < kMaxK / kWave; ++e) {
      const int j = e * kWave + lane;
      if (e * kWave >= a.k) continue;
      const float p = exp2_split(lp[e]);
      S += p;
      if (j < a.k) {
        sp[j] = p;
        slp[j] = lp[e];
      }
    }
    S = wave_sum(S);
    if (__ballot(bad)) S = __builtin_nanf("");
    if (lane == 0) sS = S;
  }
  float X, S;
  row_sums(r, a.c, tid, sums, X, S, [](float) {});
  if constexpr (NT == kWave) __syncthreads();
  const float mass = sS;
  const bool none = mass == 0.f;  // no entry, or none with any weight
  if constexpr (kGrad) {
    uint16_t* drow = a.dz + row * a.ldd;
    // q_v S_t scale T, in the two forms that the sums take (an infinite X has but the second)
    const bool far = is_far(X, a.c);
    const float off = X * a.c;
    const float w = mass * a.grad / S;
    const float wn = w * fast_exp2(__builtin_fmaf(-X, a.c, off));
    auto write = [&](auto f) __attribute__((always_inline)) {
      r.vectors(tid, [&](const u32x4& v, int i, int) {
        u32x4 o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = pack_bf16x2(f(bf16_lo(v[q])), f(bf16_hi(v[q])));
        if (a.same_phase) {
          __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(drow + r.head) + i);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) drow[r.head + i * 8 + e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
        }
      });
      if (r.eidx >= 0) drow[r.eidx] = f32_to_bf16(f(r.xe));
    };
    auto near_x = [&](float x) __attribute__((always_inline)) { return fast_exp2(__builtin_fmaf(x, a.c, -off)) * wn; };
    auto far_x = [&](float x) __attribute__((always_inline)) { return fast_exp2((x - X) * a.c) * w; };
    if (none) write([](float) { return 0.f; });  // whatever the row holds
    else if (!far) write(near_x);
    else write(far_x);
    if (!none) {
      // The k entries again, with their p taken off before the one rounding: the first
      // of equal ids adds up all of them, in a fixed order. A few threads share an entry.
      __syncthreads();
      int per = 1;
      while (per < 16 && a.k * per * 2 <= NT) per *= 2;
      for (int j = tid / per; j < a.k; j += NT / per) {
        const int id = sid[j];
        float p = 0.f;
        int lead = a.k;
        for (int i = tid % per; i < a.k; i += per)
          if (sid[i] == id) {
            lead = min(lead, i);
            p += sp[i];
          }
        for (int o = 1; o < per; o <<= 1) {
          lead = min(lead, __shfl_xor(lead, o, kWave));
          p += __shfl_xor(p, o, kWave);
        }
        if (tid % per == 0 && id >= 0 && lead == j)
          drow[id] = f32_to_bf16((far ? far_x(sz[j]) : near_x(sz[j])) - p * a.grad);
      }
    }
  }
  if (tid < kWave) {
    const double l2 = log2((double)S);  // of the sum against X, which comes off each logit first
    double sum = 0.0;
    for (int j = lane; j < a.k; j += kWave) {
      const float p = sp[j];
      if (p != 0.f) sum += (double)p * (slp[j] - (((double)sz[j] - (double)X) * (double)a.c - l2));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if (lane == 0) a.loss[row] = none ? 0.f : (mass != mass ? mass : (float)(sum * (double)a.t2ln2));
  }
}

// Threads and vectors per thread for a row of V elements (a workgroup holds 8 NT NVEC
// of them, less up to 7 before the first vector): the fewest threads whose registers
// hold the row, so that several rows share a CU and one's loads pass under another's
// sums. Rows of up to 2055 logits take one wave and no barrier (16384 x 500, k = 64:
// 44 us, with 4 waves 330); 1024 threads for 50257 logits took 844 us where 512 took 482.
#define NL_ROW_SIZES(X) X(64, 1) X(64, 2) X(64, 4) X(256, 2) X(512, 2) X(512, 4) X(512, 7) X(512, 10) X(512, 13) X(1024, 9) X(1024, 13)

// threads of a row's workgroup
int row_threads(int V) {
#define NL_THREADS(NT, NV) \
  if (V / 8 <= NT * NV) return NT;
  NL_ROW_SIZES(NL_THREADS)
#undef NL_THREADS
  return 1024;
}

void launch_top(hipStream_t st, int M, int V, const uint16_t* x, int64_t ld, int k, float t, uint16_t* values,
                int32_t* ids, float* lse) {
  const float c = kLog2e / t;
  const double inv_t = 1.0 / t;
#define NL_TOP(NT, NV)                                                                                           \
  if (V / 8 <= NT * NV) {                                                                                        \
    hipLaunchKernelGGL((top_kernel<NT, NV>), dim3(M), dim3(NT), 0, st, V, x, ld, k, c, inv_t, values, ids, lse); \
    return;                                                                                                      \
  }
  NL_ROW_SIZES(NL_TOP)
#undef NL_TOP
  hipLaunchKernelGGL((top_kernel<1024, 0>), dim3(M), dim3(1024), 0, st, V, x, ld, k, c, inv_t, values, ids, lse);
}

template <bool kGrad>
void launch_distill(hipStream_t st, int M, const DistillArgs& a) {
#define NL_DISTILL(NT, NV)                                                                     \
  if (a.V / 8 <= NT * NV) {                                                                    \
    hipLaunchKernelGGL((distill_kernel<NT, NV, kGrad>), dim3(M), dim3(NT), 0, st, a);          \
    return;                                                                                    \
  }
  NL_ROW_SIZES(NL_DISTILL)
#undef NL_DISTILL
  hipLaunchKernelGGL((distill_kernel<1024, 0, kGrad>), dim3(M), dim3(1024), 0, st, a);
}

int check_rows(const char* what, int M, int V, const void* logits, int64_t ld, int k, float t) {
  const std::string w(what);
  if (M < 0 || V <= 0 || V >= (1 << 24)) return nl_set_error(NL_EINVAL, w + ": need M >= 0 and 0 < V < 2^24");
  if (k < 1 || k > kMaxK) return nl_set_error(NL_EINVAL, w + ": need 1 <= k <= NL_TOP_MAX_K");
  if (!(t > 0.f) || t == INFINITY || !(kLog2e / t < INFINITY) || !(t * t < INFINITY) || kLog2e / t < 1e-30f)
    return nl_set_error(NL_EINVAL, w + ": the temperature must be positive and finite");
  if ((int64_t)M * row_threads(V) >= (int64_t)1 << 32)  // the threads of one launch
    return nl_set_error(NL_EUNSUPPORTED, w + ": too many rows");
  if (M > 0 && !logits) return nl_set_error(NL_EINVAL, w + ": null logits");
  if (M > 1 && ld < V) return nl_set_error(NL_EINVAL, w + ": ld < V");
  if ((uintptr_t)logits & 1) return nl_set_error(NL_EALIGN, w + ": logits not 2-byte aligned");
  return NL_OK;
}

}  // namespace
}  // namespace nl

using namespace nl;

extern "C" int nl_top_logits(void* stream, int M, int V, const nl_bf16* logits, int64_t ld, int k, float temperature,
                             nl_bf16* values, int32_t* ids, float* lse) {
  if (int rc = check_rows("top_logits", M, V, logits, ld, k, temperature)) return rc;
  if (k > V) return nl_set_error(NL_EINVAL, "top_logits: k > V");
  if (M == 0) return NL_OK;
  if (!values || !ids || !lse) return nl_set_error(NL_EINVAL, "top_logits: null output");
  launch_top((hipStream_t)stream, M, V, logits, ld, k, temperature, values, ids, lse);
  return nl_check_launch("nl_top_logits");
}

extern "C" int nl_distill_fwd_bwd(void* stream, int M, int V, const nl_bf16* logits, int64_t ld, int k,
                                  const void* ids, int ids_64, const void* values, int values_dtype, const float* lse,
                                  float temperature, float* loss, float* mean, float scale, nl_bf16* dlogits,
                                  int64_t ld_dlogits) {
  if (int rc = check_rows("distill", M, V, logits, ld, k, temperature)) return rc;
  if (values_dtype != NL_DTYPE_F32 && values_dtype != NL_DTYPE_BF16)
    return nl_set_error(NL_EINVAL, "distill: values are fp32 or bf16");
  if (M == 0) return mean ? nl_mean_f32(stream, loss, 0, mean) : NL_OK;
  if (!ids || !values || !loss) return nl_set_error(NL_EINVAL, "distill: null pointer");
  if (dlogits) {
    if (M > 1 && ld_dlogits < V) return nl_set_error(NL_EINVAL, "distill: ld_dlogits < V");
    if ((uintptr_t)dlogits & 1) return nl_set_error(NL_EALIGN, "distill: dlogits not 2-byte aligned");
    if ((const void*)dlogits == (const void*)logits && M > 1 && ld_dlogits != ld)
      return nl_set_error(NL_EINVAL, "distill: dlogits over the logits need ld_dlogits == ld");
  }
  DistillArgs a{V, k, logits, ld, ids, ids_64 != 0, values, values_dtype == NL_DTYPE_F32, lse,
                1.0 / temperature, kLog2e / temperature,
                temperature * temperature * kLn2, scale * temperature, loss, dlogits, ld_dlogits,
                (((uintptr_t)logits ^ (uintptr_t)dlogits) & 15) == 0 && (M == 1 || (ld - ld_dlogits) % 8 == 0)};
  if (dlogits) launch_distill<true>((hipStream_t)stream, M, a);
  else launch_distill<false>((hipStream_t)stream, M, a);
  if (int rc = nl_check_launch("nl_distill_fwd_bwd")) return rc;
  return mean ? nl_mean_f32(stream, loss, M, mean) : NL_OK;
}
