// Layer norm and RMS norm over the channels of a row, forward and backward (kg_layer_norm, kg_layer_norm_backward).
//
// With h = (x - mean) rstd: y = h gamma + beta; backward, with d = dy gamma, dx = rstd (d - mean(d) - h mean(d h)) over the
// row's channels, dgamma = sum of dy h and dbeta = sum of dy over the rows. RMS norm has no mean, in either direction.
//
// The variance comes from the deviations d from the mean as a float sum gives it. Where that mean is far from 0, their own mean says
// what its rounding left, and is taken out of both (correction).
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "kgx_device.h"
#include "kgx_learn.h"
#include "kgx_rows.h"

namespace kgx {

namespace {

constexpr int LT = 256;        // threads of a workgroup
constexpr int kMostParts = 1024;  // of the rows, for the sums over them
constexpr int kGrid = 2048;       // workgroups that take the rows in turn

struct LayerArgs {
  const void *x, *dy;
  void *y, *dx;
  long long ldx, ldy, lddy, lddx;
  const float *gamma, *beta;
  float *mean, *rstd, *dgamma, *dbeta;
  float* parts;  // [parts][2][channels] sums of dy h and dy over a part's rows
  struct RowMeans* means;  // [rows], of wide rows
  int rows, channels, rms, past, split;
  double eps, inverse;  // inverse: 1 / channels
  float shrink;         // of the elements in a sum for the mean: below 1 / channels, a power of 2, which changes no bit but an exponent's
  double grow;          // 1 / (shrink channels)
};

// The mean from the sum of elements times shrink, which is in float's range as they are. (Rounded, the mean of elements near the range's end
// may lie past it.)
__device__ __forceinline__ float mean_of(const LayerArgs& a, double sum) {
  const float mean = (float)(sum * a.grow);
  return isinf(mean) && !isinf(sum) ? copysignf(FLT_MAX, mean) : mean;
}

// (NaN stays NaN: a comparison, not fmax.)
__device__ __forceinline__ float root_of(double variance, double eps) { return (float)(1.0 / sqrt((variance < 0.0 ? 0.0 : variance) + eps)); }

// The deviations' mean where it says something of the row's mean. Below 2^-22 of their size it is their own rounding: values on a
// coarse grid less a mean off that grid are rounded the same way all over a binade (2047 rows of 10007 f16 whose mean was 0.01 of
// their size: the means were off by 4e-6 with it, by 8e-8 without).
__device__ __forceinline__ double correction(double off, double squares) { return off * off > 0x1p-44 * squares ? off : 0.0; }

// ---- Rows that fit the registers of their lanes: one read. ----

// L lanes a row: neighbours of one wave (several rows a wave below 64), or a workgroup. Lane i holds chunks i, i + L, ... of 16
// bytes. A chunk that reaches over the row's end is its last 16 bytes instead, so that no lane takes single elements: what it has of the
// chunk before counts there alone (first), and is stored twice, with the same values. Rows shorter than a chunk are taken by elements;
// in the places behind them is 0, or the row's first element (FIRST).
template <typename T, int L, int E>
struct Row {
  static constexpr int V = kVec<T>, THREADS = L <= 64 ? LT : L, ROWS = THREADS / L;  // of a workgroup
  typedef typename AnyWords<T>::type words_t;
  static __device__ __forceinline__ int lane() { return threadIdx.x % L; }
  static __device__ __forceinline__ int column(int e) { return (lane() + e * L) * V; }
  static __device__ __forceinline__ int start(int channels, int e) { return max(min(column(e), channels - V), 0); }
  // Of a lane's chunk, elements [first, limit) count; every one where whole (the same for all lanes).
  static __device__ __forceinline__ int first(int channels, int e) { return column(e) - start(channels, e); }
  static __device__ __forceinline__ int limit(int channels) { return min(channels, V); }
  static __device__ __forceinline__ bool whole(int channels, int e) { return (e + 1) * L * V <= channels; }
  enum Behind { ZERO, FIRST };
  static __device__ __forceinline__ void load(const T* row, int channels, bool in, u32x4 (&raw)[E], Behind behind = ZERO) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      raw[e] = u32x4{0, 0, 0, 0};
      if (!in) continue;
      if (channels >= V) {
        raw[e] = *(const words_t*)(row + start(channels, e));
      } else {
        unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < V; j++)
          if (j < channels || behind == FIRST) {
            const int k = j < channels ? j : 0;
            if constexpr (sizeof(T) == 4) w[j] = ((const unsigned*)row)[k];
            else w[j >> 1] |= (unsigned)((const unsigned short*)row)[k] << (j & 1 ? 16 : 0);
          }
        raw[e] = u32x4{w[0], w[1], w[2], w[3]};
      }
    }
  }
  static __device__ __forceinline__ void store(T* row, int channels, int e, bool past, const float (&f)[V]) {
    if (column(e) >= channels) return;
    T* p = row + start(channels, e);
    if (channels >= V) {
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
      for (int j = 0; j < V - 1; j++)
        if (j < channels) p[j] = to_t<T>(f[j]);
    }
  }
  // A lane's share of a vector of the channels, `none` where there is no vector.
  static __device__ __forceinline__ void vector(const float* p, int channels, float none, float (&f)[E][V]) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int c = start(channels, e);
      if (p && channels >= V) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const f32x4_any w = *(const f32x4_any*)(p + c + j);
#pragma unroll
          for (int k = 0; k < 4; k++) f[e][j + k] = w[k];
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) f[e][j] = p && j < channels ? p[j] : none;
      }
    }
  }
  // Sums over the row, in each of its lanes. red: of the workgroup, another one from call to call in turns of two or more.
  template <int N>
  static __device__ __forceinline__ void sum(float (&v)[N], float (*red)[N]) {
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = share_sum(v[k], L < 64 ? L : 64);
    if constexpr (L > 64) {
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < N; k++) red[threadIdx.x >> 6][k] = v[k];
      lds_barrier();
#pragma unroll
      for (int k = 0; k < N; k++) {
        float t[L / 64];
#pragma unroll
        for (int w = 0; w < L / 64; w++) t[w] = red[w][k];
#pragma unroll
        for (int o = L / 128; o >= 1; o >>= 1)
#pragma unroll
          for (int w = 0; w < o; w++) t[w] += t[w + o];
        v[k] = t[0];
      }
    }
  }
};

template <typename T, int L, int E>
__global__ __launch_bounds__((Row<T, L, E>::THREADS)) void layer_norm_held_kernel(LayerArgs a) {
  using R = Row<T, L, E>;
  constexpr int V = R::V;
  __shared__ float red[2][16][1], red2[2][16][2];
  float gamma[E][V], beta[E][V];
  R::vector(a.gamma, a.channels, 1.f, gamma);
  R::vector(a.beta, a.channels, 0.f, beta);
  int turn = 0;
  for (int first = blockIdx.x * R::ROWS; first < a.rows; first += gridDim.x * R::ROWS) {
    const int row = first + threadIdx.x / L;
    const bool in = row < a.rows;
    u32x4 raw[E];
    R::load((const T*)a.x + (size_t)row * a.ldx, a.channels, in, raw);
    float mean = 0.f;
    if (!a.rms) {
      float s[1] = {0.f};
#pragma unroll
      for (int e = 0; e < E; e++) {
        const bool whole = R::whole(a.channels, e);
        const int least = R::first(a.channels, e), limit = R::limit(a.channels);
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) t = __builtin_fmaf(whole || (j >= least && j < limit) ? element<T>(raw[e], j) : 0.f, a.shrink, t);
        s[0] += t;
      }
      R::sum(s, red[turn]);
      mean = mean_of(a, (double)s[0]);
    }
    float q[2] = {0.f, 0.f};  // of the deviations, and of their squares
#pragma unroll
    for (int e = 0; e < E; e++) {
      const bool whole = R::whole(a.channels, e);
      const int least = R::first(a.channels, e), limit = R::limit(a.channels);
      float t = 0.f, u = 0.f;
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float d = whole || (j >= least && j < limit) ? element<T>(raw[e], j) - mean : 0.f;
        t += d;
        u = __builtin_fmaf(d, d, u);
      }
      q[0] += t;
      q[1] += u;
    }
    R::sum(q, red2[turn]);
    turn ^= 1;
    const double squares = (double)q[1] * a.inverse, m = a.rms ? 0.0 : correction((double)q[0] * a.inverse, squares);
    const float rstd = root_of(squares - m * m, a.eps), shift = (float)m;
    if (!in) continue;
    T* y = (T*)a.y + (size_t)row * a.ldy;
#pragma unroll
    for (int e = 0; e < E; e++) {
      float f[V];
#pragma unroll
      for (int j = 0; j < V; j++) f[j] = __builtin_fmaf(((element<T>(raw[e], j) - mean) - shift) * rstd, gamma[e][j], beta[e][j]);
      R::store(y, a.channels, e, a.past, f);
    }
    if (R::lane() == 0) {
      if (!a.rms) a.mean[row] = (float)((double)mean + m);
      a.rstd[row] = rstd;
    }
  }
}

// Forward, a workgroup a row: its chunks lie along the lines of y (see Chunks), so that rows of odd strides are stored in whole ones, and
// gamma and beta are read where they are used, which leaves a CU's registers to four rows and more: 2047 rows of 10007 f16 take
// 22 us among other calls, 23 to 28 in a graph by how many buffers take turns (94 with chunks from the row's start and gamma and beta in registers, one row a CU).
template <typename T, int NT, int E>
__global__ __launch_bounds__(NT) void layer_norm_wide_kernel(LayerArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float red[2][16][1], red2[2][16][2];
  typedef Row<T, NT, E> R;
  const int tid = threadIdx.x;
  int turn = 0;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + (size_t)row * a.ldx;
    T* y = (T*)a.y + (size_t)row * a.ldy;
    const Chunks<T> at(a.channels, y);
    u32x4 raw[E];
    load_row<T, NT, E>(x, tid, at, raw);
    float mean = 0.f;
    if (!a.rms) {
      float s[1] = {0.f};
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (at.none(e * NT)) break;
        const int c = tid + e * NT, first = at.first(c), limit = at.limit(c);
        float t = 0.f;
        if (at.whole(e * NT, NT)) {
#pragma unroll
          for (int j = 0; j < V; j++) t = __builtin_fmaf(element<T>(raw[e], j), a.shrink, t);
        } else {
#pragma unroll
          for (int j = 0; j < V; j++) t = __builtin_fmaf(j >= first && j < limit ? element<T>(raw[e], j) : 0.f, a.shrink, t);
        }
        s[0] += t;
      }
      R::sum(s, red[turn]);
      mean = mean_of(a, (double)s[0]);
    }
    forget<E>(raw);
    float q[2] = {0.f, 0.f};  // of the deviations, and of their squares
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (at.none(e * NT)) break;
      const int c = tid + e * NT, first = at.first(c), limit = at.limit(c);
      const bool whole = at.whole(e * NT, NT);
      float t = 0.f, u = 0.f;
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float d = whole || (j >= first && j < limit) ? element<T>(raw[e], j) - mean : 0.f;
        t += d;
        u = __builtin_fmaf(d, d, u);
      }
      q[0] += t;
      q[1] += u;
    }
    R::sum(q, red2[turn]);
    turn ^= 1;
    const double squares = (double)q[1] * a.inverse, m = a.rms ? 0.0 : correction((double)q[0] * a.inverse, squares);
    const float rstd = root_of(squares - m * m, a.eps), shift = (float)m;
    forget<E>(raw);
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (at.none(e * NT)) break;
      const int c = fresh(tid) + e * NT, start = at.start(c);
      float f[V];
#pragma unroll
      for (int j = 0; j < V; j++) f[j] = ((element<T>(raw[e], j) - mean) - shift) * rstd;
      if (a.gamma) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const f32x4_any w = *(const f32x4_any*)(a.gamma + start + j);
#pragma unroll
          for (int k = 0; k < 4; k++) f[j + k] *= w[k];
        }
      }
      if (a.beta) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const f32x4_any w = *(const f32x4_any*)(a.beta + start + j);
#pragma unroll
          for (int k = 0; k < 4; k++) f[j + k] += w[k];
        }
      }
      store_gradient<T>(y, c, at.whole(e * NT, NT), a.past, at, f);
    }
    if (tid == 0) {
      if (!a.rms) a.mean[row] = (float)((double)mean + m);
      a.rstd[row] = rstd;
    }
  }
}

// Backward, the rows of a workgroup one after another, with the channels' sums of dy h and dy in registers: a part for each workgroup.
// Here for rows of a wave and less.
template <typename T, int L, int E>
__global__ __launch_bounds__(LT) void layer_norm_back_held_kernel(LayerArgs a) {
  using R = Row<T, L, E>;
  constexpr int V = R::V, SPAN = L * E * V;  // elements that a row's lanes hold
  __shared__ float joined[2 * SPAN];
  float gamma[E][V], s1[E][V] = {}, s2[E][V] = {};
  R::vector(a.gamma, a.channels, 1.f, gamma);
  for (int first = blockIdx.x * R::ROWS; first < a.rows; first += gridDim.x * R::ROWS) {
    const int row = first + threadIdx.x / L;
    const bool in = row < a.rows;
    u32x4 x[E], dy[E];
    R::load((const T*)a.x + (size_t)row * a.ldx, a.channels, in, x, R::FIRST);
    R::load((const T*)a.dy + (size_t)row * a.lddy, a.channels, in, dy);
    const float mean = a.rms || !in ? 0.f : a.mean[row], rstd = in ? a.rstd[row] : 0.f;
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; e++) {
      const bool whole = R::whole(a.channels, e);
      const int least = R::first(a.channels, e);
      float t = 0.f, u = 0.f;
#pragma unroll
      for (int j = 0; j < V; j++) {
        // (Behind a short row's end dy is 0 and h is an element's: of 0 less a large mean it would be infinite, and their product NaN.)
        const float g = whole || j >= least ? element<T>(dy[e], j) : 0.f, d = g * gamma[e][j], h = (element<T>(x[e], j) - mean) * rstd;
        t += d;
        u = __builtin_fmaf(d, h, u);
        s1[e][j] = __builtin_fmaf(g, h, s1[e][j]);
        s2[e][j] += g;
      }
      q[0] += t;
      q[1] += u;
    }
    R::sum(q, (float(*)[2])nullptr);
    if (!in) continue;
    const float m1 = a.rms ? 0.f : (float)((double)q[0] * a.inverse), m2 = (float)((double)q[1] * a.inverse);
    T* dx = (T*)a.dx + (size_t)row * a.lddx;
    if constexpr (E > 1) {
      forget<E>(x);
      forget<E>(dy);
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
      float f[V];
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float d = element<T>(dy[e], j) * gamma[e][j], h = (element<T>(x[e], j) - mean) * rstd;
        f[j] = rstd * __builtin_fmaf(-h, m2, d - m1);
      }
      R::store(dx, a.channels, e, a.past, f);
    }
  }
  if (!a.dgamma && !a.dbeta) return;
  float* part = a.parts + (size_t)blockIdx.x * 2 * a.channels;
  // The rows that a wave held side by side, then its waves in turn.
#pragma unroll
  for (int e = 0; e < E; e++) {
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
      for (int o = L; o < 64; o <<= 1) {
        s1[e][j] += __shfl_xor(s1[e][j], o);
        s2[e][j] += __shfl_xor(s2[e][j], o);
      }
    }
  }
  for (int w = 0; w < LT / 64; w++) {
    if (threadIdx.x >> 6 == w && (threadIdx.x & 63) < L) {
#pragma unroll
      for (int e = 0; e < E; e++) {
#pragma unroll
        for (int j = 0; j < V; j++) {
          if (j < R::first(a.channels, e)) continue;
          float* at = joined + R::start(a.channels, e) + j;
          at[0] = (w ? at[0] : 0.f) + s1[e][j];
          at[SPAN] = (w ? at[SPAN] : 0.f) + s2[e][j];
        }
      }
    }
    lds_barrier();
  }
  for (int c = threadIdx.x; c < a.channels; c += LT) {
    part[c] = joined[c];
    part[a.channels + c] = joined[SPAN + c];
  }
}

// The same for a workgroup a row. gamma lies in LDS, and the next row's words are asked for before this one's sums, as few workgroups
// fit a CU beside the channels' sums (12207 rows of 4096 bf16: 72 us, 85 with gamma in registers and a row at a time).
template <typename T, int NT, int E>
__global__ __launch_bounds__(NT) void layer_norm_back_wide_kernel(LayerArgs a) {
  using R = Row<T, NT, E>;
  constexpr int V = R::V;
  extern __shared__ __align__(16) float gamma[];  // [chunks][V], as the threads hold them
  __shared__ float red[2][16][2];
  float s1[E][V] = {}, s2[E][V] = {};
#pragma unroll
  for (int e = 0; e < E; e++)
    for (int j = 0; j < V; j++) gamma[(threadIdx.x + e * NT) * V + j] = a.gamma ? a.gamma[R::start(a.channels, e) + j] : 1.f;
  const auto vec4 = [&](int e, int j) { return *(const floatx4*)(gamma + (threadIdx.x + e * NT) * V + j); };
  int turn = 0;
  u32x4 x[E], dy[E], next_x[E], next_dy[E];
  const auto ask = [&](int row, u32x4(&to_x)[E], u32x4(&to_dy)[E]) {
    R::load((const T*)a.x + (size_t)row * a.ldx, a.channels, row < a.rows, to_x);
    R::load((const T*)a.dy + (size_t)row * a.lddy, a.channels, row < a.rows, to_dy);
  };
  ask(blockIdx.x, x, dy);
  __syncthreads();
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.rms ? 0.f : a.mean[row], rstd = a.rstd[row];
    ask(row + gridDim.x, next_x, next_dy);
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; e++) {
      const bool whole = R::whole(a.channels, e);
      const int least = R::first(a.channels, e);
      float t = 0.f, u = 0.f;
#pragma unroll
      for (int j4 = 0; j4 < V; j4 += 4) {
        const floatx4 w = vec4(e, j4);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int j = j4 + k;
          const float g = whole || j >= least ? element<T>(dy[e], j) : 0.f, d = g * w[k], h = (element<T>(x[e], j) - mean) * rstd;
          t += d;
          u = __builtin_fmaf(d, h, u);
          s1[e][j] = __builtin_fmaf(g, h, s1[e][j]);
          s2[e][j] += g;
        }
      }
      q[0] += t;
      q[1] += u;
      __builtin_amdgcn_sched_barrier(0);
    }
    R::sum(q, red[turn]);
    turn ^= 1;
    const float m1 = a.rms ? 0.f : (float)((double)q[0] * a.inverse), m2 = (float)((double)q[1] * a.inverse);
    T* dx = (T*)a.dx + (size_t)row * a.lddx;
    forget<E>(x);
    forget<E>(dy);
#pragma unroll
    for (int e = 0; e < E; e++) {
      float f[V];
#pragma unroll
      for (int j4 = 0; j4 < V; j4 += 4) {
        const floatx4 w = vec4(e, j4);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int j = j4 + k;
          const float d = element<T>(dy[e], j) * w[k], h = (element<T>(x[e], j) - mean) * rstd;
          f[j] = rstd * __builtin_fmaf(-h, m2, d - m1);
        }
      }
      R::store(dx, a.channels, e, a.past, f);
      x[e] = next_x[e];
      dy[e] = next_dy[e];
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (!a.dgamma && !a.dbeta) return;
  float* part = a.parts + (size_t)blockIdx.x * 2 * a.channels;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int c = R::start(a.channels, e);
#pragma unroll
    for (int j = 0; j < V; j++)
      if (j >= R::first(a.channels, e)) {
        part[c + j] = s1[e][j];
        part[a.channels + c + j] = s2[e][j];
      }
  }
}

// ---- Any row. ----

// A workgroup a row, whatever its width.
template <typename T>
__global__ __launch_bounds__(LT) void layer_norm_kernel(LayerArgs a) {
  __shared__ float red[16];
  const int tid = threadIdx.x;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + (size_t)row * a.ldx;
    T* y = (T*)a.y + (size_t)row * a.ldy;
    float mean = 0.f;
    if (!a.rms) {
      float sum = 0.f;
      for (int c = tid; c < a.channels; c += LT) sum = __builtin_fmaf((float)x[c], a.shrink, sum);
      mean = mean_of(a, row_sum<LT>(sum, red));
    }
    float off = 0.f, square = 0.f;
    for (int c = tid; c < a.channels; c += LT) {
      const float d = (float)x[c] - mean;
      off += d;
      square = __builtin_fmaf(d, d, square);
    }
    const double squares = row_sum<LT>(square, red) * a.inverse;
    const double m = a.rms ? 0.0 : correction(row_sum<LT>(off, red) * a.inverse, squares);
    const float rstd = root_of(squares - m * m, a.eps), shift = (float)m;
    for (int c = tid; c < a.channels; c += LT) {
      const float h = (((float)x[c] - mean) - shift) * rstd;
      y[c] = to_t<T>(__builtin_fmaf(h, a.gamma ? a.gamma[c] : 1.f, a.beta ? a.beta[c] : 0.f));
    }
    if (tid == 0) {
      if (!a.rms) a.mean[row] = (float)((double)mean + m);
      a.rstd[row] = rstd;
    }
  }
}

// Backward, any row: a launch for the rows' two means, by a workgroup a row, and one by slabs of the channels, whose waves take a slab of 64
// chunks over the rows in turn with the channels' sums in few registers. x and dy are read twice, in two streams without a wait between
// a row's loads and its stores.
struct RowMeans {
  float mean, rstd, m1, m2;
};
template <typename T>
__global__ __launch_bounds__(LT) void layer_norm_back_means_kernel(LayerArgs a) {
  constexpr int V = kVec<T>, E = 4;
  __shared__ float red[2][16][2];
  const int tid = threadIdx.x;
  int turn = 0;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + (size_t)row * a.ldx;
    const T* dy = (const T*)a.dy + (size_t)row * a.lddy;
    const float mean = a.rms ? 0.f : a.mean[row], rstd = a.rstd[row];
    float q[2] = {0.f, 0.f};
    for (int c0 = 0; c0 < a.channels; c0 += LT * E * V) {
      float fx[E][V], fy[E][V];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int c = min(c0 + (tid + e * LT) * V, a.channels - V);
        load_vec<T>(x + c, V, fx[e]);
        load_vec<T>(dy + c, V, fy[e]);
      }
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int c = min(c0 + (tid + e * LT) * V, a.channels - V), least = c0 + (tid + e * LT) * V - c;  // (see Row)
        float t = 0.f, u = 0.f;
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          float w[4] = {1.f, 1.f, 1.f, 1.f};
          if (a.gamma) load_vec<float>(a.gamma + c + j, 4, w);
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float d = j + k >= least ? fy[e][j + k] * w[k] : 0.f;
            t += d;
            u = __builtin_fmaf(d, (fx[e][j + k] - mean) * rstd, u);
          }
        }
        q[0] += t;
        q[1] += u;
      }
    }
    Row<T, LT, 1>::sum(q, red[turn]);
    turn ^= 1;
    if (tid == 0) a.means[row] = RowMeans{mean, rstd, a.rms ? 0.f : (float)((double)q[0] * a.inverse), (float)((double)q[1] * a.inverse)};
  }
}

constexpr int SW = LT / 64;  // waves of a slab's workgroup
template <typename T>
__global__ __launch_bounds__(LT) void layer_norm_back_slab_kernel(LayerArgs a, int slabs) {
  constexpr int V = kVec<T>, AT_ONCE = 4;
  __shared__ float joined[SW][2][64 * V];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = blockIdx.x / slabs, column = ((blockIdx.x - part * slabs) * 64 + lane) * V;
  const int c = min(column, a.channels - V), least = column - c;  // (see Row)
  const int per = (a.rows + a.split - 1) / a.split, first = part * per, last = min(first + per, a.rows);
  float gamma[V], s1[V] = {}, s2[V] = {};
#pragma unroll
  for (int j = 0; j < V; j++) gamma[j] = a.gamma ? a.gamma[c + j] : 1.f;
  for (int row = first + w; row < last; row += SW * AT_ONCE) {
    float x[AT_ONCE][V], dy[AT_ONCE][V];
#pragma unroll
    for (int k = 0; k < AT_ONCE; k++) {
      const int r = min(row + k * SW, last - 1);
      load_vec<T>((const T*)a.x + (size_t)r * a.ldx + c, V, x[k]);
      load_vec<T>((const T*)a.dy + (size_t)r * a.lddy + c, V, dy[k]);
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; k++) {
      const int r = row + k * SW;
      if (r >= last) break;
      const RowMeans n = a.means[r];
      float f[V];
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float g = dy[k][j], h = (x[k][j] - n.mean) * n.rstd;
        s1[j] = __builtin_fmaf(g, h, s1[j]);
        s2[j] += g;
        f[j] = n.rstd * __builtin_fmaf(-h, n.m2, g * gamma[j] - n.m1);
      }
      T* to = (T*)a.dx + (size_t)r * a.lddx + c;
      if (least >= V) continue;
      if (a.past) store_past<T>(to, f);
      else store_vec<T>(to, V, f);
    }
  }
  if (!a.dgamma && !a.dbeta) return;
#pragma unroll
  for (int j = 0; j < V; j++) {
    joined[w][0][lane * V + j] = s1[j];
    joined[w][1][lane * V + j] = s2[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * 64 * V; i += LT) {
    const int side = i >= 64 * V, at = i - side * 64 * V, wanted = (blockIdx.x - part * slabs) * 64 * V + at / V * V;
    const int from = min(wanted, a.channels - V);
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < SW; k++) t += joined[k][side][at];
    if (at % V >= wanted - from) a.parts[((size_t)part * 2 + side) * a.channels + from + at % V] = t;
  }
}

// The parts' sums joined in double: a workgroup takes 64 of the sums, PG groups of 16 threads the parts in turn.
constexpr int PT = 1024, PG = PT / 16;
__global__ __launch_bounds__(PT) void layer_norm_params_kernel(LayerArgs a) {
  __shared__ double joined[PG][65];
  const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
  for (long long first = blockIdx.x * 64ll; first < 2ll * a.channels; first += gridDim.x * 64ll) {
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    const long long at = first + lane * 4;
#pragma unroll 4
    for (int p = group; p < a.split; p += PG) {
      float f[4];
      load_vec<float>(a.parts + (size_t)p * 2 * a.channels + at, (int)max(min(2ll * a.channels - at, 4ll), 0ll), f);
#pragma unroll
      for (int j = 0; j < 4; j++) s[j] += (double)f[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++) joined[group][lane * 4 + j] = s[j];
    __syncthreads();
    if (threadIdx.x < 64) {
      double t = 0.0;
#pragma unroll 8
      for (int g = 0; g < PG; g++) t += joined[g][threadIdx.x];
      const long long i = first + threadIdx.x;
      float* out = i < a.channels ? a.dgamma : a.dbeta;
      if (out && i < 2ll * a.channels) out[i < a.channels ? i : i - a.channels] = (float)t;
    }
  }
}

// ---- Launches. ----

// How a row lies: L lanes with E chunks each; lanes 0 where no variant holds it.
struct Shape {
  int lanes = 0, each = 0;
};
// Forward, whose wide rows' chunks may begin up to a line before the row. (Narrow rows share a wave, so that its lanes are busy and their
// sums take fewer steps.)
template <typename T>
Shape forward_shape(const LayerArgs& p) {
  const int line = Chunks<T>::line(p.channels);
  const bool aligned = (uintptr_t)p.y % line == 0 && (p.rows == 1 || p.ldy * (long long)sizeof(T) % line == 0);
  const int least = (int)(((long long)p.channels + kVec<T> - 1) / kVec<T>), chunks = least + (aligned ? 0 : line / 16);
  if (least <= 8) return {8, 1};
  if (least <= 64) return {16, (least + 15) / 16};
  if (least <= 256) return {64, (least + 63) / 64};
  if (chunks <= 512) return {256, 2};
  if (chunks <= 1024) return {256, 4};
  if (chunks <= 2048) return {512, 4};
  if (chunks <= 4096) return {1024, 4};
  return {};
}
// Backward: few chunks a thread, whose sums of dy h and dy take four registers an element of 16 bits and more (97656 rows of 512 bf16
// by 16 lanes with four chunks: 64 us, by 64 with one 49). Wider rows go by slabs (see layer_norm_back_slab_kernel): held, a row and its
// channels' sums leave a CU one workgroup (3051 rows of 16384 bf16: 152 us, by slabs 84; 6103 of 8192 bf16 109 and 86; rows of as many
// floats hold half the sums and stay: 3051 of 8192 f32 59).
Shape backward_shape(int channels, int vec) {
  const int chunks = (int)(((long long)channels + vec - 1) / vec);
  if (chunks <= 8) return {8, 1};
  if (chunks <= 16) return {16, 1};
  if (chunks <= 32) return {32, 1};
  if (chunks <= 64) return {64, 1};
  if (chunks <= 128) return {64, 2};
  if (chunks <= 256) return {256, 1};
  if (chunks <= 512) return {256, 2};
  if (vec == 4 && chunks <= 1024) return {512, 2};
  if (vec == 4 && chunks <= 2048) return {1024, 2};
  return {};
}

// (Rows that may go by slabs, whatever their type, have their means in front of the parts.)
size_t means_bytes(int rows, int channels) { return channels > 512 * 8 ? ((size_t)rows * sizeof(RowMeans) + 255) / 256 * 256 : 0; }
// Workgroups of the backward pass, each with a part of the sums: at least eight rows each once there is one for each CU.
int parts_of(int rows, int per) { return (int)std::min((rows + (long long)per - 1) / per, (long long)std::min(std::max(256, rows / 8), kMostParts)); }

// The same by slabs: some 2048 workgroups in all, of 16 rows and more.
int slab_parts(int rows, int slabs) { return std::max(1, std::min({rows / 16, 2048 / slabs, 256})); }

LayerArgs args_of(const kg_layer_norm_args& a) {
  LayerArgs p;
  p.x = a.x; p.ldx = a.ldx;
  p.y = a.y; p.ldy = a.ldy;
  p.dy = a.dy; p.lddy = a.lddy;
  p.dx = a.dx; p.lddx = a.lddx;
  p.gamma = a.gamma; p.beta = a.beta;
  p.mean = a.mean; p.rstd = a.rstd;
  p.dgamma = a.dgamma; p.dbeta = a.dbeta;
  p.parts = (float*)((char*)a.workspace + means_bytes(a.rows, a.channels));
  p.means = (RowMeans*)a.workspace;
  p.rows = a.rows; p.channels = a.channels; p.rms = a.rms != 0;
  p.past = gradient_past(a.rows, a.channels, a.type);
  p.split = 0;
  p.eps = a.eps;
  p.inverse = 1.0 / a.channels;
  p.shrink = (float)std::ldexp(0.5, -(int)std::ceil(std::log2((double)a.channels)));
  p.grow = p.inverse / (double)p.shrink;
  return p;
}

template <typename T, int L, int E>
void forward_held(const LayerArgs& p, hipStream_t s) {
  launch_k(layer_norm_held_kernel<T, L, E>, dim3(std::min(row_grid(p.rows, Row<T, L, E>::ROWS), kGrid)), LT, 0, s, p);
}
template <typename T>
void forward_typed(const LayerArgs& p, hipStream_t s) {
  const Shape r = forward_shape<T>(p);
  const dim3 grid(row_grid(p.rows, 1));
  if (r.lanes == 8) forward_held<T, 8, 1>(p, s);
  else if (r.lanes == 16 && r.each == 1) forward_held<T, 16, 1>(p, s);
  else if (r.lanes == 16 && r.each == 2) forward_held<T, 16, 2>(p, s);
  else if (r.lanes == 16 && r.each == 3) forward_held<T, 16, 3>(p, s);
  else if (r.lanes == 16) forward_held<T, 16, 4>(p, s);
  else if (r.lanes == 64 && r.each == 2) forward_held<T, 64, 2>(p, s);
  else if (r.lanes == 64 && r.each == 3) forward_held<T, 64, 3>(p, s);
  else if (r.lanes == 64) forward_held<T, 64, 4>(p, s);
  else if (r.lanes == 256 && r.each == 2) launch_k(layer_norm_wide_kernel<T, 256, 2>, grid, 256, 0, s, p);
  else if (r.lanes == 256) launch_k(layer_norm_wide_kernel<T, 256, 4>, grid, 256, 0, s, p);
  else if (r.lanes == 512) launch_k(layer_norm_wide_kernel<T, 512, 4>, grid, 512, 0, s, p);
  else if (r.lanes == 1024) launch_k(layer_norm_wide_kernel<T, 1024, 4>, grid, 1024, 0, s, p);
  else launch_k(layer_norm_kernel<T>, grid, LT, 0, s, p);
}

template <typename T, int NT, int E>
void backward_wide(const LayerArgs& p, hipStream_t s) {
  launch_k(layer_norm_back_wide_kernel<T, NT, E>, dim3(p.split), NT, (size_t)NT * E * kVec<T> * 4, s, p);
}

// Returns the parts that the sums over the rows are in.
template <typename T>
int backward_typed(LayerArgs p, hipStream_t s) {
  const Shape r = backward_shape(p.channels, kVec<T>);
  p.split = parts_of(p.rows, r.lanes == 0 || r.lanes > 64 ? 1 : LT / r.lanes);
  const dim3 grid(p.split);
  if (r.lanes == 8) launch_k(layer_norm_back_held_kernel<T, 8, 1>, grid, LT, 0, s, p);
  else if (r.lanes == 16) launch_k(layer_norm_back_held_kernel<T, 16, 1>, grid, LT, 0, s, p);
  else if (r.lanes == 32) launch_k(layer_norm_back_held_kernel<T, 32, 1>, grid, LT, 0, s, p);
  else if (r.lanes == 64 && r.each == 1) launch_k(layer_norm_back_held_kernel<T, 64, 1>, grid, LT, 0, s, p);
  else if (r.lanes == 64) launch_k(layer_norm_back_held_kernel<T, 64, 2>, grid, LT, 0, s, p);
  else if (r.lanes == 256 && r.each == 1) backward_wide<T, 256, 1>(p, s);
  else if (r.lanes == 256) backward_wide<T, 256, 2>(p, s);
  else if (r.lanes) {
    if constexpr (sizeof(T) == 4) {
      if (r.lanes == 512) backward_wide<T, 512, 2>(p, s);
      else backward_wide<T, 1024, 2>(p, s);
    }
  } else {
    const int slabs = (int)(((long long)p.channels + 64 * kVec<T> - 1) / (64 * kVec<T>));
    p.split = slab_parts(p.rows, slabs);
    launch_k(layer_norm_back_means_kernel<T>, dim3(row_grid(p.rows, 1)), LT, 0, s, p);
    launch_k(layer_norm_back_slab_kernel<T>, dim3(p.split * slabs), LT, 0, s, p, slabs);
  }
  return p.split;
}

}  // namespace

size_t layer_norm_workspace(int rows, int channels) {
  if (rows < 1 || channels < 1) return 0;
  return means_bytes(rows, channels) + (size_t)parts_of(rows, 1) * 2 * channels * sizeof(float);
}

void launch_layer_norm(const kg_layer_norm_args& a, hipStream_t s) {
  const LayerArgs p = args_of(a);
  switch (a.type) {
    case PREC_F32: forward_typed<float>(p, s); break;
    case PREC_F16: forward_typed<f16>(p, s); break;
    default: forward_typed<bf16>(p, s); break;
  }
  KGX_CHECK_LAUNCH();
}

void launch_layer_norm_backward(const kg_layer_norm_args& a, hipStream_t s) {
  LayerArgs p = args_of(a);
  if (p.rows) {  // (the sums over no rows are 0)
    switch (a.type) {
      case PREC_F32: p.split = backward_typed<float>(p, s); break;
      case PREC_F16: p.split = backward_typed<f16>(p, s); break;
      default: p.split = backward_typed<bf16>(p, s); break;
    }
  }
  if (p.dgamma || p.dbeta) launch_k(layer_norm_params_kernel, dim3((int)std::min((2ll * p.channels + 63) / 64, 65536ll)), PT, 0, s, p);
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
