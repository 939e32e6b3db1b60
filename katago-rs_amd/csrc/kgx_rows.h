// Rows of logits in chunks of 16 bytes, for the losses: loads and stores at any alignment, the columns that take no part, sums
// and maxima over a row, and how many threads and parts a row takes.
#pragma once
#include <algorithm>
#include <climits>

#include "kgx_device.h"
#include "kgx_vec.h"
#include "kgx_wave.h"

namespace kgx {

// 16 bytes of a row at its elements' alignment: rows of odd strides and columns of a larger row start anywhere. (Global
// loads and stores of any width need no more than that on this hardware.)
typedef unsigned int u32x4_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x4_any4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct AnyWords { typedef u32x4_any2 type; };
template <> struct AnyWords<float> { typedef u32x4_any4 type; };
typedef unsigned int u32_any __attribute__((aligned(1)));
typedef unsigned long long u64_any __attribute__((aligned(1)));

// Reductions over the NT threads of a row: a wave, or the whole workgroup through `red` (16 floats).
template <int NT, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
  v = wave_reduce<MAX>(v);
  if constexpr (NT > 64) {
    lds_barrier();  // (the last reduction's values have been read)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    lds_barrier();
    v = red[0];
#pragma unroll
    for (int k = 1; k < NT / 64; k++) v = MAX ? fmaxf(v, red[k]) : v + red[k];
  }
  return v;
}

// A row's sum, its waves' added in double: a workgroup's last roundings to float are the whole sum's, and a sequence's
// log-probability adds up those of all its rows (margins of 512 rows off by 1.0e-7 rms with them, 0.4e-7 without).
template <int NT>
__device__ __forceinline__ double row_sum(float v, float* red) {
  v = wave_reduce<false>(v);
  if constexpr (NT == 64) return (double)v;
  lds_barrier();  // (the last reduction's values have been read)
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  lds_barrier();
  double t = (double)red[0];
#pragma unroll
  for (int k = 1; k < NT / 64; k++) t += (double)red[k];
  return t;
}

// log(s) in double for s >= 1, from s = 2^k f, f in [0.7, 1.42): log f = 2 atanh(t) = 2 (t + t^3/3 + ...),
// t = (f - 1) / (f + 1), |t| < 0.172, so that the terms to t^13 leave 1e-12. NaN stays; s is finite
// (a sum of at most 2^30 terms up to 1).
__device__ __forceinline__ double log_sum(double s) {
  int k;
  double f = frexp(s, &k);
  if (f < 0.70710678) { f *= 2.0; k--; }
  const double t = (f - 1.0) / (f + 1.0), q = t * t;
  double p = 1.0 / 13;
  p = __builtin_fma(p, q, 1.0 / 11);
  p = __builtin_fma(p, q, 1.0 / 9);
  p = __builtin_fma(p, q, 1.0 / 7);
  p = __builtin_fma(p, q, 1.0 / 5);
  p = __builtin_fma(p, q, 1.0 / 3);
  p = __builtin_fma(p, q, 1.0);
  return __builtin_fma((double)k, 0.69314718055994530942, 2.0 * t * p);
}

// s log2 e in two floats: the first alone is off by up to 2^-23, relative, the same way in every term of a row. A sequence's
// log-probability sums that error over its rows, and the margin is a small difference of such sums (0.15 of 5000 in a case of
// 500 tokens: the margin was off by 7e-6, with both parts by 4e-7). The first is the largest float below the product, so that the
// second is positive: both products of -infinity, which stands in every place that takes no part, are then -infinity, and never
// infinity less infinity. (s is in [2^-64, 2^64]: neither part is subnormal.) The gradients, which no sum takes further, make do
// with the first part: off by up to 2^-23 X of a probability that lies X octaves below the row's largest.
struct Base2 {
  float hi, lo;
  __device__ __forceinline__ explicit Base2(double s) {
    const double all = s * 1.44269504088896340736;
    hi = (float)all;
    if ((double)hi >= all) hi = __uint_as_float(__float_as_uint(hi) - 1);
    lo = (float)(all - (double)hi);
  }
};
// (0 below 2^-126: the hardware's exponential gives no subnormal numbers.)
__device__ __forceinline__ float exp_of(float x, Base2 c) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(x, c.hi, x * c.lo));
}

// The running maximum and sum of e^((z - top) s) over a thread's share of a row.
struct Running {
  float top = -INFINITY, sum = 0.f;
  double total = 0.0;  // the row's, once joined
  // Takes V values, which become z - top; e: their exponentials. Returns what the sum so far was scaled by, and in `moved`
  // how far the maximum it is relative to went down (old minus new).
  template <int V>
  __device__ __forceinline__ float add(float (&z)[V], Base2 c, float (&e)[V], float& moved) {
    float t = z[0];
#pragma unroll
    for (int j = 1; j < V; j++) t = fmaxf(t, z[j]);
    const float up = fmaxf(top, t);
    // (Nothing but -infinity so far: keep the sums at 0 rather than take -infinity from itself.)
    const float base = up == -INFINITY ? 0.f : up;
    moved = top - base;
    const float keep = exp_of(moved, c);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < V; j++) {
      z[j] -= base;
      e[j] = exp_of(z[j], c);
      s += e[j];
    }
    sum = __builtin_fmaf(sum, keep, s);
    top = up;
    return keep;
  }
  template <int V>
  __device__ __forceinline__ void add(float (&z)[V], Base2 c) {
    float e[V], moved;
    add<V>(z, c, e, moved);
  }
  template <int NT>
  __device__ __forceinline__ float join(Base2 c, float* red, float& moved) {  // over the row; returns as add does
    const float all = row_reduce<NT, true>(top, red);
    moved = top - all;
    const float keep = top == -INFINITY ? 0.f : exp_of(moved, c);
    total = row_sum<NT>(sum * keep, red);
    top = all;
    return keep;
  }
};

// Which of a workgroup's rows this thread's is, in a scalar register where a row is a wave.
template <int NT>
__device__ __forceinline__ int wave_row() {
  static_assert(NT == 64 || NT >= 256, "a wave a row, or a workgroup");
  return NT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
}

// Gradients of more bytes than this are stored past the caches, which then keep logits for the second reading and no lines
// that a later launch has to write back: 4093 x 32768 bf16 106 -> 97 us, 8192 x 32768 preference rows 200 -> 174. Smaller ones
// stay where the next operator finds them.
inline constexpr long long kPastBytes = 64ll << 20;

// ---- Rows that fit the registers of their threads: one read. ----

// A row's chunks of 16 bytes, laid so that `along`, the row that is written (or else read), has them at multiples of 16 bytes,
// and in rows from 4 KB on the first at a multiple of 128, so that a wave's chunks are whole cache lines: chunk c is elements
// [c V - back, (c + 1) V - back) of the row, back the elements from such a multiple to its start. (Rows of odd strides: stores
// across 16 bytes cost a quarter of the time over 2700 x 100003 f16, and parts of lines a tenth when stored past the
// caches.) A chunk that reaches over either end of the row, and one past the end, is read from the row's first or last 16
// bytes instead, so that no load is behind a branch: of what is read there, elements [first, limit) are the chunk's.
template <typename T>
struct Chunks {
  static constexpr int V = kVec<T>;
  int columns, back;
  __device__ __forceinline__ Chunks(int columns_, const T* along)
      : columns(columns_), back(__builtin_amdgcn_readfirstlane((int)((uintptr_t)along & (line(columns_) - 1)) / (int)sizeof(T))) {}
  static __host__ __device__ __forceinline__ int line(int columns) { return columns < 4096 / (int)sizeof(T) ? 16 : 128; }
  __device__ __forceinline__ int start(int c) const { return max(min(c * V - back, columns - V), 0); }
  __device__ __forceinline__ int first(int c) const { return min(max(c * V - back - start(c), 0), V); }
  __device__ __forceinline__ int limit(int c) const { return min((c + 1) * V - back - start(c), V); }
  __device__ __forceinline__ int of(int column) const { return (column + back) / V; }
  __device__ __forceinline__ bool none(int c) const { return c * V - back >= columns; }                  // c and all behind it
  __device__ __forceinline__ bool whole(int c, int n) const { return c * V >= back && (c + n) * V - back <= columns; }  // n from c on
};

template <typename T>
__device__ __forceinline__ float element(const u32x4& w, int j) {
  if constexpr (std::is_same<T, float>::value) {
    return __uint_as_float(w[j]);
  } else {
    const unsigned x = w[j >> 1];
    if constexpr (std::is_same<T, bf16>::value) return __uint_as_float(j & 1 ? x & 0xffff0000u : x << 16);
    else return (float)__builtin_bit_cast(f16, (unsigned short)(j & 1 ? x >> 16 : x));
  }
}
// -infinity in the place of element j.
template <typename T>
__device__ __forceinline__ void remove(u32x4& w, int j, bool gone) {
  if constexpr (std::is_same<T, float>::value) {
    w[j] = gone ? 0xff800000u : w[j];
  } else {
    constexpr unsigned inf = std::is_same<T, bf16>::value ? 0xff80u : 0xfc00u;
    const unsigned x = w[j >> 1];
    w[j >> 1] = gone ? (j & 1 ? (x & 0xffffu) | inf << 16 : (x & 0xffff0000u) | inf) : x;
  }
}
template <typename T>
__device__ __forceinline__ u32x4 words_of(const float (&f)[kVec<T>]) {
  u32x4 w;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    if constexpr (std::is_same<T, float>::value) w[k] = __float_as_uint(f[k]);
    else w[k] = __builtin_bit_cast(unsigned short, to_t<T>(f[2 * k])) | (unsigned)__builtin_bit_cast(unsigned short, to_t<T>(f[2 * k + 1])) << 16;
  }
  return w;
}
// Makes the words new to the compiler: what was computed from them before is computed again rather than kept in registers.
template <int E>
__device__ __forceinline__ void forget(u32x4 (&raw)[E]) {
#pragma unroll
  for (int e = 0; e < E; e++) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      unsigned w = raw[e][k];
      asm("" : "+v"(w));
      raw[e][k] = w;
    }
  }
}
// A value that the compiler takes for new: what follows from it is computed here rather than kept over the loop of rows.
__device__ __forceinline__ int fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
template <typename T, int NT, int E>
__device__ __forceinline__ void load_row(const T* row, int tid, const Chunks<T>& at, u32x4 (&raw)[E], int c0 = 0) {
  tid = fresh(tid + c0);
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (at.none(c0 + e * NT)) break;  // (here and below: no thread has such a chunk)
    raw[e] = *(const typename AnyWords<T>::type*)(row + at.start(tid + e * NT));
  }
}
template <typename T, int NT, int E>
__device__ __forceinline__ void remove_past(int tid, const Chunks<T>& at, u32x4 (&raw)[E], int c0 = 0) {
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (at.none(c0 + e * NT)) break;
    if (at.whole(c0 + e * NT, NT)) continue;
    const int c = fresh(tid) + c0 + e * NT, first = at.first(c), limit = at.limit(c);
    if (first > 0 || limit < kVec<T>) {
#pragma unroll
      for (int j = 0; j < kVec<T>; j++) remove<T>(raw[e], j, j < first || j >= limit);
    }
    __builtin_amdgcn_sched_barrier(0);  // (here and below: a chunk at a time, so that registers hold little beside the row)
  }
}
// -infinity in the place of illegal elements, of the row and of the reference's (where FULL).
template <typename T, int NT, int E, bool FULL>
__device__ __forceinline__ void remove_illegal(const unsigned char* legal, int tid, const Chunks<T>& at, u32x4 (&raw)[E],
                                               u32x4 (&ref)[FULL ? E : 1], int c0 = 0) {
  constexpr int V = kVec<T>;
  unsigned long long ok[E];
  const int t = fresh(tid + c0);
#pragma unroll
  for (int e = 0; e < E; e++) {
    ok[e] = ~0ull;
    if (at.none(c0 + e * NT)) continue;
    const unsigned char* p = legal + at.start(t + e * NT);
    if constexpr (V == 4) ok[e] = *(const u32_any*)p;
    else ok[e] = *(const u64_any*)p;
  }
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (at.none(c0 + e * NT)) break;
#pragma unroll
    for (int j = 0; j < V; j++) {
      const bool gone = ((ok[e] >> (8 * j)) & 0xff) == 0;
      remove<T>(raw[e], j, gone);
      if constexpr (FULL) remove<T>(ref[e], j, gone);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <typename T, int NT, int E>
__device__ __forceinline__ float max_of(const u32x4 (&raw)[E], const Chunks<T>& at, float* red) {
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (at.none(e * NT)) break;
#pragma unroll
    for (int j = 0; j < kVec<T>; j++) top = fmaxf(top, element<T>(raw[e], j));
    __builtin_amdgcn_sched_barrier(0);
  }
  return row_reduce<NT, true>(top, red);
}
// past: past the caches (kPastBytes).
template <typename T>
__device__ __forceinline__ void store_gradient(T* row, int c, bool whole, bool past, const Chunks<T>& at, const float (&f)[kVec<T>]) {
  typedef typename AnyWords<T>::type words_t;
  const int first = whole ? 0 : at.first(c), limit = whole ? kVec<T> : at.limit(c);
  T* p = row + at.start(c);
  if (whole || (first == 0 && limit == kVec<T>)) {
    const words_t w = words_of<T>(f);
    if (past) {
      asm volatile("");  // (or the two stores become one, a plain one)
      __builtin_nontemporal_store(w, (words_t*)p);
      asm volatile("");
    } else {
      *(words_t*)p = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kVec<T>; j++)
      if (j >= first && j < limit) p[j] = to_t<T>(f[j]);
  }
}

// Workgroups of a launch over rows, `per` at a time: the grid's threads stay below 2^32 and each workgroup strides on.
inline int row_grid(int rows, int per) {
  const long long n = ((long long)rows + per - 1) / per;
  return (int)(n < (1 << 20) ? n : (1 << 20));
}

// The threads and chunks a thread of a row of `columns` elements of 16 / vec bytes that stays in registers; threads 0 where it
// does not fit: a row shorter than a chunk, or longer than 4096 chunks. A wave a row up to 512 chunks needs no barrier;
// beyond, the fewest threads that hold it in 8 chunks each.
// (Rows that do not start at a line's multiple may reach into as many chunks more as a line has.)
struct RowShape {
  int threads = 0, each = 0;
};
template <typename T>
RowShape row_shape(int columns, const void* p, long long ld, int rows) {
  constexpr int vec = kVec<T>;
  const int line = Chunks<T>::line(columns);
  const bool aligned = (uintptr_t)p % line == 0 && (rows == 1 || ld * (long long)sizeof(T) % line == 0);
  const int chunks = (int)(((long long)columns + vec - 1) / vec) + (aligned ? 0 : line / 16);
  if (columns < vec || chunks > 4096) return {};
  if (chunks <= 128) return {64, 2};
  if (chunks <= 512) return {64, 8};
  if (chunks <= 2048) return {256, 8};
  return {512, 8};
}

// How many parts a row may be cut into, four workgroups a CU in all: what the workspace holds. (257 rows of 100003 bf16 with a full
// KL 88 us whole, 63 in parts; 512 rows 133 and 114, but 27 and 34 of 40001 without a reference.)
inline int most_parts(int rows, int columns) { return rows < 1 || rows > 384 || columns <= 16384 ? 1 : std::min(64, 1024 / rows); }

// The parts that a call takes, of whole pieces of `piece` chunks each.
struct RowParts {
  int split, span;
};
template <typename T>
RowParts row_parts(int rows, int columns, int piece) {
  const int chunks = (columns + kVec<T> - 1) / kVec<T> + Chunks<T>::line(columns) / 16, pieces = (chunks + piece - 1) / piece;
  const int most = std::min(most_parts(rows, columns), pieces), each = (pieces + most - 1) / most;
  return {(pieces + each - 1) / each, each * piece};
}

inline bool gradient_past(int rows, int columns, int type) { return (long long)rows * columns * (type == PREC_F32 ? 4 : 2) > kPastBytes; }

}  // namespace kgx
