// Group norm with an activation on channels-last rows under the board mask, forward and backward (kg_group_norm,
// kg_group_norm_backward).
//
// Bound by memory: x read and y written once, or dy and x read and dx written once.
// - Where a slab of whole groups over all points of a batch row fits the registers of one workgroup (up to 128 KB: the
//   boards of every network here, images of 64 x 64), it is read once, the statistics meet in LDS, and the result is
//   written from the registers. Slabs are narrow, so that few rows fill the chip; neighbouring slabs, which share cache lines,
//   run on one XCD.
// - Longer rows are cut into shares of the points: the same slabs, once for their part of the statistics and once for the
//   result, whose second reading comes from the caches where they fit.
// - Channels fewer than a 16-byte column's, and groups wider than a workgroup joins, go by rows: simple kernels that take any
//   width.
// A thread keeps its column of 16 bytes for all its points.
#include <algorithm>

#include "kgx_device.h"
#include "kgx_learn.h"
#include "kgx_wave.h"

namespace kgx {

namespace {

constexpr int GT = 256;         // threads of a workgroup
constexpr int kSplitTarget = 16384;  // elements a workgroup, about
constexpr int kMaxGroups = 2048;     // group statistics in LDS
constexpr int kCUs = 256;
// Results of more bytes than this are stored past the caches, which then keep x and dy for their second reading (16 x 8192
// points of 512 f32 channels forward 177 -> 131 us, of bf16 backward 138 -> 118). Smaller ones stay where the next operator
// finds them.
constexpr long long kPastBytes = 64ll << 20;

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
template <typename T> constexpr int kVec = 16 / sizeof(T);
template <typename T> struct RowVec { typedef u16x8_any type; };
template <> struct RowVec<float> { typedef f32x4_any type; };

template <typename T>
__device__ __forceinline__ float widen1(const typename RowVec<T>::type& v, int j) {
  if constexpr (std::is_same<T, float>::value) return v[j];
  else if constexpr (std::is_same<T, bf16>::value) return __uint_as_float((unsigned)v[j] << 16);
  else return (float)__builtin_bit_cast(f16, (unsigned short)v[j]);
}
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, int left, float (&f)[kVec<T>]) {
  if (left >= kVec<T>) {
    const typename RowVec<T>::type v = *(const typename RowVec<T>::type*)p;
#pragma unroll
    for (int j = 0; j < kVec<T>; j++) f[j] = widen1<T>(v, j);
  } else {
#pragma unroll
    for (int j = 0; j < kVec<T>; j++) f[j] = j < left ? (float)p[j] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, int left, const float (&f)[kVec<T>]) {
  T t[kVec<T>];
#pragma unroll
  for (int j = 0; j < kVec<T>; j++) t[j] = to_t<T>(f[j]);
  if (left >= kVec<T>) {
    *(typename RowVec<T>::type*)p = __builtin_bit_cast(typename RowVec<T>::type, t);
  } else {
#pragma unroll
    for (int j = 0; j < kVec<T>; j++)
      if (j < left) p[j] = t[j];
  }
}

struct NormArgs {
  const void *x, *dy;
  void *y, *dx;
  long long ldx, ldy, lddy, lddx;
  const float *mask, *gamma, *beta;
  float *mean, *rstd, *dgamma, *dbeta;
  float* part;     // forward: [batch][splits][3][groups] count, mean, M2; backward: [batch][splits][2][channels] sums
  float* counts;   // backward: [batch][splits] points
  float* sums;     // backward: [batch][splits][2][groups] sums of da gamma and da gamma xh
  float* means;    // backward by rows: [batch][2][groups]
  int batch, points, channels, groups, width, splits;  // width: channels of a group
  int slab_groups, each;  // slabs: their groups, the points a thread takes
  int past;               // y or dx is stored past the caches
  float eps;
};

// act_f, but for ReLU of NaN, which act_f makes 0: a norm with a value that is no finite number shows it in every activation.
template <int ACT>
__device__ __forceinline__ float norm_act(float v) {
  if constexpr (ACT == ACT_RELU) return v < 0.f ? 0.f : v;
  else return act_f<ACT>(v);
}

// The points [p0, p1) of split k.
__device__ __forceinline__ void split_range(const NormArgs& a, int k, int& p0, int& p1) {
  p0 = (int)((long long)a.points * k / a.splits);
  p1 = (int)((long long)a.points * (k + 1) / a.splits);
}

// How the workgroup's threads cover rows: `cols` columns of 16 bytes side by side (of the row's `total`, from `first` on),
// and `lanes` points at a time.
struct Cover {
  int cols, lanes, col, lane;
  __device__ __forceinline__ Cover(int total, int first) {
    cols = min(total - first, GT);
    lanes = GT / cols;
    col = threadIdx.x % cols;
    lane = threadIdx.x / cols;
  }
};

// Forward, first launch: count, mean and sum of squared deviations of every group over the workgroup's points. A thread
// takes kPiece points at a time relative to the mean of its points so far (of the first piece: to its first value), s1 and s2 their sum
// and sum of squares: M2 grows by s2 - s1^2 / n. A mean far from 0 does not cancel, and one value far from the rest only within
// a piece (relative to the first value throughout, 3906 points with such a first one left 7 % of an error). The parts are joined
// pairwise exactly: M2 = sum M2_i + n_i (mean_i - mean)^2.
constexpr int kPiece = 16;
template <typename T>
__global__ __launch_bounds__(GT) void norm_stats_kernel(NormArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float s_mean[GT * V], s_m2[GT * V], s_n[GT];
  __shared__ float g_n[kMaxGroups], g_mean[kMaxGroups], g_m2[kMaxGroups];
  const int b = blockIdx.x / a.splits, k = blockIdx.x % a.splits, tid = threadIdx.x;
  int p0, p1;
  split_range(a, k, p0, p1);
  const int total = (a.channels + V - 1) / V;
  for (int g = tid; g < a.groups; g += GT) g_n[g] = g_mean[g] = g_m2[g] = 0.f;
  for (int first = 0; first < total; first += GT) {
    const Cover w(total, first);
    const int c0 = (first + w.col) * V, left = a.channels - c0;
    float mean[V], m2[V], n = 0.f;
#pragma unroll
    for (int j = 0; j < V; j++) mean[j] = m2[j] = 0.f;
    if (w.lane < w.lanes) {
      const T* x = (const T*)a.x + (size_t)b * a.points * a.ldx + c0;
      for (int p = p0 + w.lane; p < p1;) {
        float s1[V], s2[V];
        const float before = n;
#pragma unroll
        for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.f;
        for (int i = 0; i < kPiece && p < p1; i++, p += w.lanes) {
          if (a.mask && a.mask[(size_t)b * a.points + p] == 0.f) continue;
          float f[V];
          load_vec<T>(x + (size_t)p * a.ldx, left, f);
          if (n == 0.f) {
#pragma unroll
            for (int j = 0; j < V; j++) mean[j] = f[j];
          }
          n += 1.f;
#pragma unroll
          for (int j = 0; j < V; j++) {
            const float d = f[j] - mean[j];
            s1[j] += d;
            s2[j] = __builtin_fmaf(d, d, s2[j]);
          }
        }
        if (n == before) continue;
        const float inv = 1.f / n;
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float up = s1[j] * inv;
          m2[j] += fmaxf(__builtin_fmaf(-s1[j], up, s2[j]), 0.f);
          mean[j] += up;
        }
      }
    }
    s_n[tid] = n;
#pragma unroll
    for (int j = 0; j < V; j++) {
      s_mean[j * GT + tid] = mean[j];
      s_m2[j * GT + tid] = m2[j];
    }
    __syncthreads();
    // Groups with channels in this column block: 256 / share groups at a time, `share` threads each.
    const int cb0 = first * V, cb1 = min(a.channels, (first + w.cols) * V);
    const int g0 = cb0 / a.width, g1 = (cb1 - 1) / a.width + 1;
    int share = 64;
    while (share > 1 && share * (g1 - g0) > GT) share >>= 1;
    const int sub = tid % share, per = GT / share;
    for (int gb = g0; gb < g1; gb += per) {
      const int g = gb + tid / share;
      const bool on = g < g1;
      const int ca = on ? max(g * a.width, cb0) - cb0 : 0, cc = on ? min((g + 1) * a.width, cb1) - cb0 - ca : 0;
      const int items = cc * w.lanes;
      float cn = 0.f, cs = 0.f;
      for (int i = sub; i < items; i += share) {
        const int c = ca + i % cc, t = (i / cc) * w.cols + c / V;
        cn += s_n[t];
        cs = __builtin_fmaf(s_n[t], s_mean[(c % V) * GT + t], cs);
      }
      for (int o = share >> 1; o >= 1; o >>= 1) { cn += __shfl_xor(cn, o); cs += __shfl_xor(cs, o); }
      const float mean = cn > 0.f ? cs / cn : 0.f;
      float m2 = 0.f;
      for (int i = sub; i < items; i += share) {
        const int c = ca + i % cc, t = (i / cc) * w.cols + c / V;
        const float d = s_mean[(c % V) * GT + t] - mean;
        m2 += s_m2[(c % V) * GT + t] + s_n[t] * d * d;
      }
      for (int o = share >> 1; o >= 1; o >>= 1) m2 += __shfl_xor(m2, o);
      if (on && sub == 0 && cn > 0.f) {  // joined with the earlier column blocks' part of the group
        const float n0 = g_n[g], n1 = n0 + cn, d = mean - g_mean[g];
        g_mean[g] += d * (cn / n1);
        g_m2[g] += m2 + d * d * (n0 * (cn / n1));
        g_n[g] = n1;
      }
    }
    __syncthreads();
  }
  float* out = a.part + (size_t)blockIdx.x * 3 * a.groups;
  for (int g = tid; g < a.groups; g += GT) {
    out[g] = g_n[g];
    out[a.groups + g] = g_mean[g];
    out[2 * a.groups + g] = g_m2[g];
  }
}

template <typename T, int ACT>
__global__ __launch_bounds__(GT) void norm_apply_kernel(NormArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float g_mean[kMaxGroups], g_rstd[kMaxGroups];
  const int b = blockIdx.x / a.splits, k = blockIdx.x % a.splits, tid = threadIdx.x;
  int p0, p1;
  split_range(a, k, p0, p1);
  int share = 64;
  while (share > 1 && share * a.groups > GT) share >>= 1;
  for (int gb = 0; gb < a.groups; gb += GT / share) {
    const int g = gb + tid / share, sub = tid % share;
    const float* in = a.part + (size_t)b * a.splits * 3 * a.groups + min(g, a.groups - 1);
    float n = 0.f, s = 0.f, m2 = 0.f;
    for (int i = sub; i < a.splits; i += share) {
      const float* q = in + (size_t)i * 3 * a.groups;
      n += q[0];
      s = __builtin_fmaf(q[0], q[a.groups], s);
    }
    for (int o = share >> 1; o >= 1; o >>= 1) { n += __shfl_xor(n, o); s += __shfl_xor(s, o); }
    const float mean = n > 0.f ? s / n : 0.f;
    for (int i = sub; i < a.splits; i += share) {
      const float* q = in + (size_t)i * 3 * a.groups;
      const float d = q[a.groups] - mean;
      m2 += q[2 * a.groups] + (q[0] > 0.f ? q[0] * d * d : 0.f);
    }
    for (int o = share >> 1; o >= 1; o >>= 1) m2 += __shfl_xor(m2, o);
    if (g < a.groups && sub == 0) {
      const float rstd = 1.f / sqrtf((n > 0.f ? m2 / n : 0.f) + a.eps);
      g_mean[g] = mean;
      g_rstd[g] = rstd;
      if (k == 0) {
        a.mean[(size_t)b * a.groups + g] = mean;
        a.rstd[(size_t)b * a.groups + g] = rstd;
      }
    }
  }
  __syncthreads();
  const int total = (a.channels + V - 1) / V;
  for (int first = 0; first < total; first += GT) {
    const Cover w(total, first);
    if (w.lane >= w.lanes) continue;
    const int c0 = (first + w.col) * V, left = a.channels - c0;
    float mean[V], mul[V], add[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int c = min(c0 + j, a.channels - 1), g = c / a.width;
      mean[j] = g_mean[g];
      mul[j] = g_rstd[g] * (a.gamma ? a.gamma[c] : 1.f);
      add[j] = a.beta ? a.beta[c] : 0.f;
    }
    const T* x = (const T*)a.x + (size_t)b * a.points * a.ldx + c0;
    T* y = (T*)a.y + (size_t)b * a.points * a.ldy + c0;
    for (int p = p0 + w.lane; p < p1; p += w.lanes) {
      float f[V];
      if (a.mask && a.mask[(size_t)b * a.points + p] == 0.f) {
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = 0.f;
      } else {
        load_vec<T>(x + (size_t)p * a.ldx, left, f);
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = norm_act<ACT>(__builtin_fmaf(f[j] - mean[j], mul[j], add[j]));
      }
      store_vec<T>(y + (size_t)p * a.ldy, left, f);
    }
  }
}

// d act(a) / d a. Mish: with e = exp(a) and n = e (e + 2), tanh(softplus) = n / (n + 2) and 1 - tanh^2 = 4 (e + 1)^2 /
// (n + 2)^2, so the derivative n / (n + 2) + 4 a e (e + 1) / (n + 2)^2 has no cancellation but its own sign's. From a = 20 on
// it is 1 in float, as it is at 20: the argument is held there, with no branch. The exponentials are the fast ones, off by some U |a|
// (U = 2^-24) of terms that fall as a e^-|a|: a few U of the slope, as the reciprocals' ulp.
template <int ACT>
__device__ __forceinline__ float act_slope(float v) {
  if constexpr (ACT == ACT_RELU) {
    return v > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == ACT_MISH) {
    const float u = fminf(v, 20.f), e = __expf(u), n = e * (e + 2.f), r = __builtin_amdgcn_rcpf(n + 2.f);
    return n * r + 4.f * u * (e * r) * ((e + 1.f) * r);
  } else if constexpr (ACT == ACT_SILU) {
    const float q = __builtin_amdgcn_rcpf(1.f + __expf(-v));
    return q * (1.f + v * (1.f - q));
  } else {
    return 1.f;
  }
}

// A column's parameters in the backward pass, and with xc = x - mean (xh = xc rstd) the gradient at the norm's output: da =
// dy act'(xh gamma + beta). The channels' sums are taken of da xc and multiplied by rstd at the end: three values a channel
// in registers rather than four (128 KB of 16-bit x and dy leave no more).
template <typename T, int ACT, int V = kVec<T>>
struct BackColumn {
  static constexpr bool kExactSide = ACT == ACT_RELU && sizeof(T) == 4;
  float mean[V], mul[V], beta[V];
  double scale[kExactSide ? V : 1];
  __device__ __forceinline__ void load(const NormArgs& a, int b, int c0) {
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int c = min(c0 + j, a.channels - 1), g = c / a.width;
      const float rstd = a.rstd[(size_t)b * a.groups + g], gamma = a.gamma ? a.gamma[c] : 1.f;
      mean[j] = a.mean[(size_t)b * a.groups + g];
      mul[j] = rstd * gamma;
      beta[j] = a.beta ? a.beta[c] : 0.f;
      if constexpr (kExactSide) scale[j] = (double)rstd * (double)gamma;
    }
  }
  // The same from a slab's copy in LDS, in column order.
  __device__ __forceinline__ void read(const float* c_mean, const float* c_mul, const float* c_beta, const double* c_scale, int c) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const floatx4 m = *(const floatx4*)(c_mean + c + j), u = *(const floatx4*)(c_mul + c + j), t = *(const floatx4*)(c_beta + c + j);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        mean[j + k] = m[k];
        mul[j + k] = u[k];
        beta[j + k] = t[k];
        if constexpr (kExactSide) scale[j + k] = c_scale[c + j + k];
      }
    }
  }
  __device__ __forceinline__ void grad(float x, float dy, int j, float& xc, float& da) const {
    xc = x - mean[j];
    if constexpr (kExactSide) {
      // The side of 0 in double: a float's rounding there would switch a whole gradient.
      da = __builtin_fma((double)x - (double)mean[j], scale[j], (double)beta[j]) > 0.0 ? dy : 0.f;
    } else {
      da = dy * act_slope<ACT>(__builtin_fmaf(xc, mul[j], beta[j]));
    }
  }
};

// What dx takes besides: dx = rstd (da gamma - m1 - xh m2) = da mul - k1 - xc k2, with m1 and m2 the group's means of da gamma
// and da gamma xh.
__device__ __forceinline__ float back_dx(float da, float xc, float mul, float k1, float k2) {
  return __builtin_fmaf(da, mul, __builtin_fmaf(-xc, k2, -k1));
}

// Backward, first launch: sums of da and da xh over the workgroup's points, per channel, and with gamma per group.
template <typename T, int ACT>
__global__ __launch_bounds__(GT) void norm_back_sums_kernel(NormArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float s_b[GT * V], s_g[GT * V], s_n[GT];
  const int b = blockIdx.x / a.splits, k = blockIdx.x % a.splits, tid = threadIdx.x;
  int p0, p1;
  split_range(a, k, p0, p1);
  const int total = (a.channels + V - 1) / V;
  float* out = a.part + (size_t)blockIdx.x * 2 * a.channels;
  for (int first = 0; first < total; first += GT) {
    const Cover w(total, first);
    const int c0 = (first + w.col) * V, left = a.channels - c0;
    float sb[V], sg[V], n = 0.f;
#pragma unroll
    for (int j = 0; j < V; j++) sb[j] = sg[j] = 0.f;
    if (w.lane < w.lanes) {
      BackColumn<T, ACT> col;
      col.load(a, b, c0);
      const T* x = (const T*)a.x + (size_t)b * a.points * a.ldx + c0;
      const T* dy = (const T*)a.dy + (size_t)b * a.points * a.lddy + c0;
      for (int p = p0 + w.lane; p < p1; p += w.lanes) {
        if (a.mask && a.mask[(size_t)b * a.points + p] == 0.f) continue;
        n += 1.f;
        float f[V], d[V];
        load_vec<T>(x + (size_t)p * a.ldx, left, f);
        load_vec<T>(dy + (size_t)p * a.lddy, left, d);
#pragma unroll
        for (int j = 0; j < V; j++) {
          float xc, da;
          col.grad(f[j], d[j], j, xc, da);
          sb[j] += da;
          sg[j] = __builtin_fmaf(da, xc, sg[j]);
        }
      }
    }
    s_n[tid] = n;
#pragma unroll
    for (int j = 0; j < V; j++) { s_b[j * GT + tid] = sb[j]; s_g[j * GT + tid] = sg[j]; }
    __syncthreads();
    const int here = min(a.channels - first * V, w.cols * V);
    for (int c = tid; c < here; c += GT) {
      float tb = 0.f, tg = 0.f;
      for (int l = 0; l < w.lanes; l++) {
        const int t = (c % V) * GT + l * w.cols + c / V;
        tb += s_b[t];
        tg += s_g[t];
      }
      out[first * V + c] = tb;
      out[a.channels + first * V + c] = tg * a.rstd[(size_t)b * a.groups + (first * V + c) / a.width];
    }
    if (first == 0 && tid == 0) {
      float t = 0.f;
      for (int l = 0; l < w.lanes; l++) t += s_n[l * w.cols];
      a.counts[blockIdx.x] = t;
    }
    __syncthreads();
  }
  // (The channels' sums that the workgroup has just written.)
  for (int g = tid >> 6; g < a.groups; g += GT / 64) {
    float s1 = 0.f, s2 = 0.f;
#pragma unroll 4
    for (int c = g * a.width + (tid & 63); c < (g + 1) * a.width; c += 64) {
      const float gm = a.gamma ? a.gamma[c] : 1.f;
      s1 = __builtin_fmaf(gm, out[c], s1);
      s2 = __builtin_fmaf(gm, out[a.channels + c], s2);
    }
    s1 = share_sum(s1, 64);
    s2 = share_sum(s2, 64);
    if ((tid & 63) == 0) {
      float* to = a.sums + (size_t)blockIdx.x * 2 * a.groups + g;
      to[0] = s1;
      to[a.groups] = s2;
    }
  }
}

// Second launch: a wave a group of a batch row, its sums divided by its elements.
__global__ __launch_bounds__(GT) void norm_back_join_kernel(NormArgs a) {
  const int lane = threadIdx.x & 63, id = (int)blockIdx.x * (GT / 64) + (threadIdx.x >> 6);
  if (id >= a.batch * a.groups) return;
  const int b = id / a.groups, g = id % a.groups;
  float n = 0.f, s1 = 0.f, s2 = 0.f;
  for (int k = lane; k < a.splits; k += 64) n += a.counts[(size_t)b * a.splits + k];
  for (int k = lane; k < a.splits; k += 64) {
    const float* q = a.sums + ((size_t)b * a.splits + k) * 2 * a.groups + g;
    s1 += q[0];
    s2 += q[a.groups];
  }
  n = share_sum(n, 64);
  s1 = share_sum(s1, 64);
  s2 = share_sum(s2, 64);
  if (lane == 0) {
    const float inv = n > 0.f ? 1.f / (n * (float)a.width) : 0.f;
    a.means[(size_t)b * 2 * a.groups + g] = s1 * inv;
    a.means[(size_t)b * 2 * a.groups + a.groups + g] = s2 * inv;
  }
}

// Third launch: dx.
template <typename T, int ACT>
__global__ __launch_bounds__(GT) void norm_back_apply_kernel(NormArgs a) {
  constexpr int V = kVec<T>;
  const int b = blockIdx.x / a.splits, k = blockIdx.x % a.splits;
  int p0, p1;
  split_range(a, k, p0, p1);
  const int total = (a.channels + V - 1) / V;
  for (int first = 0; first < total; first += GT) {
    const Cover w(total, first);
    if (w.lane >= w.lanes) continue;
    const int c0 = (first + w.col) * V, left = a.channels - c0;
    BackColumn<T, ACT> col;
    col.load(a, b, c0);
    float k1[V], k2[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int g = min(c0 + j, a.channels - 1) / a.width;
      const float rstd = a.rstd[(size_t)b * a.groups + g];
      k1[j] = rstd * a.means[(size_t)b * 2 * a.groups + g];
      k2[j] = rstd * rstd * a.means[(size_t)b * 2 * a.groups + a.groups + g];
    }
    const T* x = (const T*)a.x + (size_t)b * a.points * a.ldx + c0;
    const T* dy = (const T*)a.dy + (size_t)b * a.points * a.lddy + c0;
    T* dx = (T*)a.dx + (size_t)b * a.points * a.lddx + c0;
    for (int p = p0 + w.lane; p < p1; p += w.lanes) {
      float f[V];
      if (a.mask && a.mask[(size_t)b * a.points + p] == 0.f) {
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = 0.f;
      } else {
        float d[V];
        load_vec<T>(x + (size_t)p * a.ldx, left, f);
        load_vec<T>(dy + (size_t)p * a.lddy, left, d);
#pragma unroll
        for (int j = 0; j < V; j++) {
          float xc, da;
          col.grad(f[j], d[j], j, xc, da);
          f[j] = back_dx(da, xc, col.mul[j], k1[j], k2[j]);
        }
      }
      store_vec<T>(dx + (size_t)p * a.lddx, left, f);
    }
  }
}

// ---- Slabs: whole groups over the points of a batch row, or over one of its shares, in a workgroup's registers. ----

// i / n for 0 <= i < 2048 and 1 <= n <= 2048, from (i + 1/2) / n in float: its error, 2^-21 of a quotient below 2048 / n, is less
// than the half n-th that it lies from a whole number. (The compiler's division takes 30 instructions.)
__device__ __forceinline__ int part_of(int i, int n) { return (int)(((float)i + 0.5f) * __builtin_amdgcn_rcpf((float)n)); }

// A workgroup's slab: thread (col, lane) takes points p0 + lane + e lanes, e < each (at most E), of the slab's 16-byte column
// col. A last column that is not whole starts earlier: its first `skip` channels are the column's before, and both threads
// compute the same for them. Threads and points past the end read the last one's address, so that no load is behind a
// branch of its own.
template <typename T, int E>
struct Slab {
  static constexpr int V = kVec<T>;
  int b, k, c0, p0, each, threads, width, cols, lanes, col, lane, start, skip, last;  // width: the slab's channels
  unsigned in, on;  // bit e: the point exists; and is not masked
  // Neighbouring slabs (which share cache lines) are on one XCD, workgroup g running on XCD g mod 8. last_first: each XCD's
  // slabs in the other order, for a second reading that begins with what the caches still hold (16 x 4096 points of 512 f32
  // channels backward: 154 -> 134 us). False past the last.
  __device__ __forceinline__ bool take(const NormArgs& a, bool last_first = false) {
    const int slabs = a.groups / a.slab_groups, n = a.batch * a.splits * slabs, per = (n + 7) / 8;
    const int at = blockIdx.x >> 3, id = (int)(blockIdx.x & 7) * per + (last_first ? per - 1 - at : at);
    if (id >= n) return false;
    // (Scalar registers: every address is one of them plus a 32-bit offset.)
    const int row = __builtin_amdgcn_readfirstlane(id / slabs);
    c0 = __builtin_amdgcn_readfirstlane((id - row * slabs) * a.slab_groups * a.width);
    b = __builtin_amdgcn_readfirstlane(row / a.splits);
    k = row - b * a.splits;
    each = a.each;
    threads = blockDim.x;
    width = a.slab_groups * a.width;
    cols = (width + V - 1) / V;
    lanes = __builtin_amdgcn_readfirstlane(part_of(threads, cols));
    lane = part_of(threadIdx.x, cols);
    col = threadIdx.x - lane * cols;
    start = min(col * V, width - V);
    skip = col * V - start;
    p0 = k * lanes * each;
    last = min(a.points - p0, lanes * each) - 1;
    in = 0;
#pragma unroll
    for (int e = 0; e < E; e++) in |= (lane < lanes && e < each && lane + e * lanes <= last ? 1u : 0u) << e;
    on = in;
    if (a.mask) {
      const float* mask = a.mask + (size_t)b * a.points + p0;
      float mk[E];
#pragma unroll
      for (int e = 0; e < E; e++) mk[e] = mask[point(e)];
#pragma unroll
      for (int e = 0; e < E; e++) on &= ~((mk[e] == 0.f ? 1u : 0u) << e);
    }
    return true;
  }
  __device__ __forceinline__ unsigned point(int e) const { return min(lane + e * lanes, last); }
  // In column order (an entry a thread, columns * V <= threads): the channel of the slab.
  __device__ __forceinline__ int channel() const { return min((int)threadIdx.x / V * V, width - V) + (int)threadIdx.x % V; }
  // Byte offset of point e's column from the slab's first element (below 2^31: slab_shape).
  __device__ __forceinline__ unsigned at(int e, unsigned ld) const { return (point(e) * ld + start) * (unsigned)sizeof(T); }
};

// A column's 16 bytes as words; element j of them as a float, and back.
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
template <typename T>
__device__ __forceinline__ unsigned word_of(float lo, float hi) {  // (float: hi is not used)
  if constexpr (std::is_same<T, float>::value) return __float_as_uint(lo);
  else return __builtin_bit_cast(unsigned short, to_t<T>(lo)) | (unsigned)__builtin_bit_cast(unsigned short, to_t<T>(hi)) << 16;
}
template <typename T> struct AnyWords;  // 16 bytes at their elements' alignment
typedef unsigned int u32x4_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x4_any4 __attribute__((ext_vector_type(4), aligned(4)));
template <> struct AnyWords<float> { typedef u32x4_any4 type; };
template <> struct AnyWords<f16> { typedef u32x4_any2 type; };
template <> struct AnyWords<bf16> { typedef u32x4_any2 type; };

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
// Zeros in the place of points that are not `on`.
template <int E>
__device__ __forceinline__ void clear_off(u32x4 (&raw)[E], unsigned on) {
#pragma unroll
  for (int e = 0; e < E; e++) {
#pragma unroll
    for (int k = 0; k < 4; k++) raw[e][k] = on >> e & 1 ? raw[e][k] : 0u;
  }
}
template <int N>
__device__ __forceinline__ void read_lds(const float* p, float (&f)[N]) {  // (N floats at a multiple of 16 bytes)
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const floatx4 v = *(const floatx4*)(p + j);
#pragma unroll
    for (int k = 0; k < 4; k++) f[j + k] = v[k];
  }
}

// All loads of a thread's column, issued before any is used (masked points too: what they hold is not looked at).
template <typename T, int E>
__device__ __forceinline__ void load_slab(const NormArgs& a, const Slab<T, E>& s, const void* from, long long ld, u32x4 (&raw)[E]) {
  const char* base = (const char*)((const T*)from + ((size_t)s.b * a.points + s.p0) * ld + s.c0);
#pragma unroll
  for (int e = 0; e < E; e++) {
    raw[e] = u32x4{0, 0, 0, 0};
    if (e < s.each) raw[e] = *(const typename AnyWords<T>::type*)(base + s.at(e, (unsigned)ld));
  }
}
template <typename T, int E>
__device__ __forceinline__ void store_slab(const NormArgs& a, const Slab<T, E>& s, void* to, long long ld, int e, const u32x4& raw) {
  char* base = (char*)((T*)to + ((size_t)s.b * a.points + s.p0) * ld + s.c0);
  if (s.in >> e & 1) {
    auto* p = (typename AnyWords<T>::type*)(base + s.at(e, (unsigned)ld));
    if (a.past) {
      asm volatile("");  // (or the compiler makes one ordinary store of the two)
      __builtin_nontemporal_store((typename AnyWords<T>::type)raw, p);
      asm volatile("");
    } else *p = raw;
  }
}

// The lanes that share a group in a join over `groups` groups by `threads` threads (groups <= threads).
__device__ __forceinline__ int join_share(int groups, int threads) {
  int share = 64;
  while (share > 1 && share * groups > threads) share >>= 1;
  return share;
}

extern __shared__ __align__(16) float slab_lds[];
// Floats of LDS: the threads' sums (two a channel of a column, at a stride that puts a column's channels in different banks),
// later the columns' parameters; then what the joins pass on.
__host__ __device__ __forceinline__ int slab_stride(int threads) { return threads + 8; }
inline size_t slab_lds_bytes(int vec, int threads, int cols, int groups, bool backward) {
  const int sums = std::max(2 * vec * slab_stride(threads), 3 * vec * cols);
  return (size_t)(backward ? sums + 3 * threads + 2 * groups + 2 + 5 * vec * cols : sums + 4 * threads + 2 * groups) * 4;
}

// The parameters that a thread puts into LDS for all, loaded early.
struct ColumnEntry {
  bool mine;
  int group;
  float gamma, beta;
  template <typename T, int E>
  __device__ __forceinline__ ColumnEntry(const NormArgs& a, const Slab<T, E>& s) {
    mine = (int)threadIdx.x < s.cols * kVec<T>;
    const int c = mine ? s.channel() : 0;
    group = part_of(c, a.width);
    gamma = a.gamma ? a.gamma[s.c0 + c] : 1.f;
    beta = a.beta ? a.beta[s.c0 + c] : 0.f;
  }
};

// y from the words of x, with the groups' mean and rstd in LDS: the columns' parameters first (over the threads' sums, which
// have been read).
template <typename T, int ACT, int E>
__device__ __forceinline__ void slab_forward(const NormArgs& a, Slab<T, E>& s, const ColumnEntry& entry, u32x4 (&raw)[E],
                                             const float* g_mean, const float* g_rstd) {
  constexpr int V = kVec<T>;
  const int all = s.cols * V;
  float *c_mean = slab_lds, *c_mul = c_mean + all, *c_add = c_mul + all;
  if (entry.mine) {
    c_mean[threadIdx.x] = g_mean[entry.group];
    c_mul[threadIdx.x] = g_rstd[entry.group] * entry.gamma;
    c_add[threadIdx.x] = entry.beta;
  }
  __syncthreads();
  asm("" : "+v"(s.lane));  // (addresses too are computed again)
  forget<E>(raw);
  float mean[V], mul[V], add[V];
  read_lds<V>(c_mean + s.col * V, mean);
  read_lds<V>(c_mul + s.col * V, mul);
  read_lds<V>(c_add + s.col * V, add);
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (e >= s.each) break;
    float f[V];
#pragma unroll
    for (int j = 0; j < V; j++) f[j] = norm_act<ACT>(__builtin_fmaf(element<T>(raw[e], j) - mean[j], mul[j], add[j]));
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      w[k] = sizeof(T) == 4 ? word_of<T>(f[k], 0.f) : word_of<T>(f[(2 * k) % V], f[(2 * k + 1) % V]);
      w[k] = s.on >> e & 1 ? w[k] : 0u;
    }
    store_slab<T, E>(a, s, a.y, a.ldy, e, w);
  }
}

// Forward over a slab: 32 boards of 361 x 384 bf16 with mish 10.2 us (latency: two workgroups' loads, joins and stores a CU at most),
// 128 boards 27 us (2.6 TB/s; identity 23, 3.1 TB/s). PART: its groups' count, mean and squared deviations over the workgroup's share of the points, for
// norm_slab_apply_kernel; else y.
template <typename T, int ACT, int NT, int E, bool PART>
__global__ __launch_bounds__(NT) void norm_slab_kernel(NormArgs a) {
  constexpr int V = kVec<T>;
  Slab<T, E> s;
  if (!s.take(a)) return;
  const int tid = threadIdx.x, P = slab_stride(s.threads);
  float *s_mean = slab_lds, *s_m2 = s_mean + V * P, *s_n = slab_lds + max(2 * V * P, 3 * V * s.cols), *r_n = s_n + s.threads,
        *r_mean = r_n + s.threads, *r_m2 = r_mean + s.threads, *g_mean = r_m2 + s.threads, *g_rstd = g_mean + a.slab_groups;
  u32x4 raw[E];
  load_slab<T, E>(a, s, a.x, a.ldx, raw);
  const ColumnEntry entry(a, s);
  clear_off<E>(raw, s.on);

  // A thread's own count, means, and squared deviations from them.
  const float n = (float)__builtin_popcount(s.on), inv = s.on ? 1.f / n : 0.f;
  float m[V], m2[V];
#pragma unroll
  for (int j = 0; j < V; j++) m[j] = m2[j] = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (e >= s.each) break;
#pragma unroll
    for (int j = 0; j < V; j++) m[j] += element<T>(raw[e], j);
  }
#pragma unroll
  for (int j = 0; j < V; j++) m[j] *= inv;
  forget<E>(raw);
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (e >= s.each) break;
#pragma unroll
    for (int j = 0; j < V; j++) {
      const float d = s.on >> e & 1 ? element<T>(raw[e], j) - m[j] : 0.f;
      m2[j] = __builtin_fmaf(d, d, m2[j]);
    }
  }
  if (s.lane < s.lanes) {
    if (s.col == 0) s_n[s.lane] = n;
#pragma unroll
    for (int j = 0; j < V; j++)
      if (j >= s.skip) {
        s_mean[(j - s.skip) * P + tid] = m[j];
        s_m2[(j - s.skip) * P + tid] = m2[j];
      }
  }
  __syncthreads();
  // Joined over the lanes: R rows of the slab's channels, then over a group's channels and those rows. Each join is
  // exact: the mean first, then M2 = sum M2_i + n_i (mean_i - mean)^2.
  const int R = min(part_of(s.threads, s.width), s.lanes);
  if (tid < R * s.width) {
    const int r = part_of(tid, s.width), c = tid - r * s.width;
    const float* qm = s_mean + (c % V) * P + c / V;
    const float* q2 = s_m2 + (c % V) * P + c / V;
    float cn = 0.f, cs = 0.f, c2 = 0.f;
    for (int l = r; l < s.lanes; l += R) {
      cn += s_n[l];
      cs = __builtin_fmaf(s_n[l], qm[l * s.cols], cs);
    }
    const float mean = cn > 0.f ? cs / cn : 0.f;
    for (int l = r; l < s.lanes; l += R) {
      const float d = qm[l * s.cols] - mean;
      c2 += q2[l * s.cols] + s_n[l] * d * d;
    }
    r_n[tid] = cn;
    r_mean[tid] = mean;
    r_m2[tid] = c2;
  }
  __syncthreads();
  {
    const int share = join_share(a.slab_groups, s.threads), sub = tid & (share - 1), g = part_of(tid, share);
    const bool mine = g < a.slab_groups;
    const int items = mine ? a.width * R : 0, first = mine ? g * a.width : 0;
    float cn = 0.f, cs = 0.f, c2 = 0.f;
    for (int i = sub; i < items; i += share) {
      const int at = part_of(i, a.width) * (s.width - a.width) + first + i;
      cn += r_n[at];
      cs = __builtin_fmaf(r_n[at], r_mean[at], cs);
    }
    cn = share_sum(cn, share);
    cs = share_sum(cs, share);
    const float mean = cn > 0.f ? cs / cn : 0.f;
    for (int i = sub; i < items; i += share) {
      const int at = part_of(i, a.width) * (s.width - a.width) + first + i;
      const float d = r_mean[at] - mean;
      c2 += r_m2[at] + r_n[at] * d * d;
    }
    c2 = share_sum(c2, share);
    if (mine && sub == 0) {
      if constexpr (PART) {
        float* out = a.part + (size_t)(s.b * a.splits + s.k) * 3 * a.groups + s.c0 / a.width + g;
        out[0] = cn;
        out[a.groups] = mean;
        out[2 * a.groups] = c2;
      } else {
        const float rstd = 1.f / sqrtf((cn > 0.f ? c2 / cn : 0.f) + a.eps);
        g_mean[g] = mean;
        g_rstd[g] = rstd;
        const size_t out = (size_t)s.b * a.groups + s.c0 / a.width + g;
        a.mean[out] = mean;
        a.rstd[out] = rstd;
      }
    }
  }
  if constexpr (!PART) {
    __syncthreads();
    slab_forward<T, ACT, E>(a, s, entry, raw, g_mean, g_rstd);
  }
}

// y over a slab's share of the points, from the shares' statistics (a.part).
template <typename T, int ACT, int NT, int E>
__global__ __launch_bounds__(NT) void norm_slab_apply_kernel(NormArgs a) {
  Slab<T, E> s;
  if (!s.take(a, true)) return;
  const int tid = threadIdx.x;
  float *g_mean = slab_lds + 3 * kVec<T> * s.cols, *g_rstd = g_mean + a.slab_groups;
  u32x4 raw[E];
  load_slab<T, E>(a, s, a.x, a.ldx, raw);
  const ColumnEntry entry(a, s);
  const int share = join_share(a.slab_groups, s.threads), sub = tid & (share - 1), g = part_of(tid, share);
  const bool mine = g < a.slab_groups;
  const float* in = a.part + (size_t)s.b * a.splits * 3 * a.groups + s.c0 / a.width + (mine ? g : 0);
  float n = 0.f, sum = 0.f, m2 = 0.f;
  for (int i = sub; i < a.splits; i += share) {
    const float* q = in + (size_t)i * 3 * a.groups;
    n += q[0];
    sum = __builtin_fmaf(q[0], q[a.groups], sum);
  }
  n = share_sum(n, share);
  sum = share_sum(sum, share);
  const float mean = n > 0.f ? sum / n : 0.f;
  for (int i = sub; i < a.splits; i += share) {
    const float* q = in + (size_t)i * 3 * a.groups;
    const float d = q[a.groups] - mean;
    m2 += q[2 * a.groups] + (q[0] > 0.f ? q[0] * d * d : 0.f);
  }
  m2 = share_sum(m2, share);
  if (mine && sub == 0) {
    const float rstd = 1.f / sqrtf((n > 0.f ? m2 / n : 0.f) + a.eps);
    g_mean[g] = mean;
    g_rstd[g] = rstd;
    if (s.k == 0) {
      a.mean[(size_t)s.b * a.groups + s.c0 / a.width + g] = mean;
      a.rstd[(size_t)s.b * a.groups + s.c0 / a.width + g] = rstd;
    }
  }
  __syncthreads();
  slab_forward<T, ACT, E>(a, s, entry, raw, g_mean, g_rstd);
}

// The backward pass's parameters in LDS, in column order: mean, rstd gamma and beta; for float ReLU also their exact product.
struct BackLds {
  float *mean, *mul, *beta;
  double* scale;
};
template <typename T, int ACT, int E>
__device__ __forceinline__ void back_params(const NormArgs& a, const Slab<T, E>& s, const BackLds& c) {
  const ColumnEntry entry(a, s);
  if (entry.mine) {
    const int i = threadIdx.x;
    const size_t g = (size_t)s.b * a.groups + s.c0 / a.width + entry.group;
    const float rstd = a.rstd[g];
    c.mean[i] = a.mean[g];
    c.mul[i] = rstd * entry.gamma;
    c.beta[i] = entry.beta;
    if constexpr (BackColumn<T, ACT>::kExactSide) c.scale[i] = (double)rstd * (double)entry.gamma;
  }
}

// KEEP: the first pass's da stay in registers for the second (at most four points a thread). They take those of a second
// workgroup on the CU, so only launches that have none keep them: mish, 361 points of 384 bf16 channels, 32 boards 14.3 us
// and 18.0 without, 128 boards 50.4 us and 46.3.
// dx from the words of x and dy (0 at masked points; or da, KEEP), with the groups' k1 and k2 in LDS.
template <typename T, int ACT, int E, bool KEEP>
__device__ __forceinline__ void slab_backward(const NormArgs& a, Slab<T, E>& s, u32x4 (&rx)[E], u32x4 (&rd)[E],
                                              float (&da)[KEEP ? E : 1][kVec<T>], const BackLds& c, const float* g_1, const float* g_2) {
  constexpr int V = kVec<T>, H = 4;
  const int all = s.cols * V;
  float *c_k1 = slab_lds, *c_k2 = c_k1 + all;
  if ((int)threadIdx.x < all) {
    const int g = part_of(s.channel(), a.width);
    c_k1[threadIdx.x] = g_1[g];
    c_k2[threadIdx.x] = g_2[g];
  }
  __syncthreads();
  asm("" : "+v"(s.lane));  // (addresses too are computed again)
  forget<E>(rx);
  if constexpr (!KEEP) forget<E>(rd);
#pragma unroll
  for (int h = 0; h < V; h += H) {
    BackColumn<T, ACT, H> col;
    float k1[H], k2[H];
    if constexpr (KEEP) {
      read_lds<H>(c.mean + s.col * V + h, col.mean);
      read_lds<H>(c.mul + s.col * V + h, col.mul);
    } else col.read(c.mean, c.mul, c.beta, c.scale, s.col * V + h);
    read_lds<H>(c_k1 + s.col * V + h, k1);
    read_lds<H>(c_k2 + s.col * V + h, k2);
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (e >= s.each) break;
      float dx[H];
#pragma unroll
      for (int j = 0; j < H; j++) {
        float xc, d;
        if constexpr (KEEP) {
          xc = element<T>(rx[e], h + j) - col.mean[j];
          d = da[e][h + j];
        } else col.grad(element<T>(rx[e], h + j), element<T>(rd[e], h + j), j, xc, d);
        dx[j] = back_dx(d, xc, col.mul[j], k1[j], k2[j]);
      }
#pragma unroll
      for (int k = 0; k < H * (int)sizeof(T) / 4; k++)
        rd[e][h * (int)sizeof(T) / 4 + k] = sizeof(T) == 4 ? word_of<T>(dx[k], 0.f) : word_of<T>(dx[(2 * k) % H], dx[(2 * k + 1) % H]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  clear_off<E>(rd, s.on);
#pragma unroll
  for (int e = 0; e < E; e++) store_slab<T, E>(a, s, a.dx, a.lddx, e, rd[e]);
}

// Backward over a slab. The channels' sums over the workgroup's points go to part [batch][splits][2][channels] for dgamma and
// dbeta. PART: the groups' sums over them go to sums and counts for norm_back_slab_apply_kernel; else dx follows. x and dy take
// 64 of a thread's 128 registers, so a column's channels are taken four at a time with their parameters from LDS, and dx
// replaces dy in place. dy is 0 at masked points, and with it da. 128 boards of 361 x 384 bf16 with mish 45 us, 16 x 4096 points of
// 512 f16 with SiLU 75 (2.7 TB/s: a slab fills the CU, so loads and the slope's exponentials take turns).
template <typename T, int ACT, int NT, int E, bool PART, bool KEEP>
__global__ __launch_bounds__(NT) void norm_back_slab_kernel(NormArgs a) {
  constexpr int V = kVec<T>, H = 4;
  Slab<T, E> s;
  if (!s.take(a)) return;
  const int tid = threadIdx.x, P = slab_stride(s.threads), all = s.cols * V;
  float *s_b = slab_lds, *s_g = s_b + V * P, *c_mean = slab_lds + max(2 * V * P, 3 * all), *s_n = c_mean + 3 * all,
        *r_b = s_n + s.threads, *r_g = r_b + s.threads, *g_1 = r_g + s.threads, *g_2 = g_1 + a.slab_groups;
  // (An even number of floats lies before it: threads and all are even, and the groups come twice.)
  const BackLds c = {c_mean, c_mean + all, c_mean + 2 * all, (double*)(g_2 + a.slab_groups)};
  u32x4 rx[E], rd[E];
  load_slab<T, E>(a, s, a.x, a.ldx, rx);
  load_slab<T, E>(a, s, a.dy, a.lddy, rd);
  back_params<T, ACT, E>(a, s, c);
  const int own = min(tid, s.width - 1), share = join_share(a.slab_groups, s.threads), sub = tid & (share - 1), g = part_of(tid, share);
  const float* rstd = a.rstd + (size_t)s.b * a.groups + s.c0 / a.width;
  const float own_rstd = rstd[part_of(own, a.width)], own_gamma = a.gamma ? a.gamma[s.c0 + own] : 1.f, g_rstd = rstd[min(g, a.slab_groups - 1)];
  if (s.lane < s.lanes && s.col == 0) s_n[s.lane] = (float)__builtin_popcount(s.on);
  lds_barrier();  // (the parameters; x and dy may still be on their way)
  clear_off<E>(rx, s.on);
  clear_off<E>(rd, s.on);
  float kept[KEEP ? E : 1][V];
#pragma unroll
  for (int h = 0; h < V; h += H) {
    BackColumn<T, ACT, H> col;
    col.read(c.mean, c.mul, c.beta, c.scale, s.col * V + h);
    float sb[H], sg[H];
#pragma unroll
    for (int j = 0; j < H; j++) sb[j] = sg[j] = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (e >= s.each) break;
#pragma unroll
      for (int j = 0; j < H; j++) {
        float xc, da;
        col.grad(element<T>(rx[e], h + j), element<T>(rd[e], h + j), j, xc, da);
        sb[j] += da;
        sg[j] = __builtin_fmaf(da, xc, sg[j]);
        if constexpr (KEEP) kept[e][h + j] = da;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (s.lane < s.lanes) {
#pragma unroll
      for (int j = 0; j < H; j++)
        if (h + j >= s.skip) {
          s_b[(h + j - s.skip) * P + tid] = sb[j];
          s_g[(h + j - s.skip) * P + tid] = sg[j];
        }
    }
  }
  __syncthreads();
  const int R = min(part_of(s.threads, s.width), s.lanes);
  if (tid < R * s.width) {
    const int r = part_of(tid, s.width), ch = tid - r * s.width, from = (ch % V) * P + ch / V;
    float tb = 0.f, tg = 0.f;
    for (int l = r; l < s.lanes; l += R) {
      tb += s_b[from + l * s.cols];
      tg += s_g[from + l * s.cols];
    }
    r_b[tid] = tb;
    r_g[tid] = tg;
  }
  __syncthreads();
  if (tid < s.width) {
    float tb = 0.f, tg = 0.f;
    for (int r = 0; r < R; r++) {
      tb += r_b[r * s.width + tid];
      tg += r_g[r * s.width + tid];
    }
    tg *= own_rstd;
    float* out = a.part + (size_t)(s.b * a.splits + s.k) * 2 * a.channels + s.c0 + tid;
    out[0] = tb;
    out[a.channels] = tg;
    s_b[tid] = tb * own_gamma;  // (the lanes' sums have been read)
    s_g[tid] = tg * own_gamma;
  }
  __syncthreads();
  const bool mine = g < a.slab_groups;
  float t1 = 0.f, t2 = 0.f, cn = 0.f;
  for (int i = sub; i < (mine ? a.width : 0); i += share) {
    t1 += s_b[g * a.width + i];
    t2 += s_g[g * a.width + i];
  }
  for (int i = sub; i < (mine ? s.lanes : 0); i += share) cn += s_n[i];
  t1 = share_sum(t1, share);
  t2 = share_sum(t2, share);
  cn = share_sum(cn, share);
  if (mine && sub == 0) {
    if constexpr (PART) {
      const size_t part = (size_t)s.b * a.splits + s.k;
      float* to = a.sums + part * 2 * a.groups + s.c0 / a.width + g;
      to[0] = t1;
      to[a.groups] = t2;
      if (s.c0 == 0 && g == 0) a.counts[part] = cn;
    } else {
      const float inv = cn > 0.f ? 1.f / (cn * (float)a.width) : 0.f;
      g_1[g] = g_rstd * (t1 * inv);
      g_2[g] = g_rstd * g_rstd * (t2 * inv);
    }
  }
  if constexpr (!PART) {
    __syncthreads();
    slab_backward<T, ACT, E, KEEP>(a, s, rx, rd, kept, c, g_1, g_2);
  }
}

// dx over a slab's share of the points, from the shares' sums (a.sums, a.counts).
template <typename T, int ACT, int NT, int E>
__global__ __launch_bounds__(NT) void norm_back_slab_apply_kernel(NormArgs a) {
  constexpr int V = kVec<T>;
  Slab<T, E> s;
  if (!s.take(a, true)) return;
  const int all = s.cols * V;
  float *c_mean = slab_lds + 3 * all, *g_1 = c_mean + 3 * all, *g_2 = g_1 + a.slab_groups;
  const BackLds c = {c_mean, c_mean + all, c_mean + 2 * all, (double*)(g_2 + a.slab_groups)};
  u32x4 rx[E], rd[E];
  load_slab<T, E>(a, s, a.x, a.ldx, rx);
  load_slab<T, E>(a, s, a.dy, a.lddy, rd);
  back_params<T, ACT, E>(a, s, c);
  const int share = join_share(a.slab_groups, s.threads), sub = threadIdx.x & (share - 1), g = part_of(threadIdx.x, share);
  const bool mine = g < a.slab_groups;
  const size_t part = (size_t)s.b * a.splits;
  const int at = s.c0 / a.width + (mine ? g : 0);
  const float rstd = a.rstd[(size_t)s.b * a.groups + at];
  float t1 = 0.f, t2 = 0.f, n = 0.f;
  for (int i = sub; i < a.splits; i += share) {
    const float* q = a.sums + (part + i) * 2 * a.groups + at;
    t1 += q[0];
    t2 += q[a.groups];
    n += a.counts[part + i];
  }
  t1 = share_sum(t1, share);
  t2 = share_sum(t2, share);
  n = share_sum(n, share);
  if (mine && sub == 0) {
    const float inv = n > 0.f ? rstd / (n * (float)a.width) : 0.f;
    g_1[g] = t1 * inv;
    g_2[g] = t2 * inv * rstd;
  }
  lds_barrier();
  clear_off<E>(rx, s.on);
  clear_off<E>(rd, s.on);
  float none[1][V];
  slab_backward<T, ACT, E, false>(a, s, rx, rd, none, c, g_1, g_2);
}

// dgamma and dbeta of 64 channels a workgroup from `parts` rows of channel sums, one wave a sixteenth of them.
__global__ __launch_bounds__(1024) void norm_back_params_kernel(NormArgs a, int parts) {
  __shared__ float red[16][2][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (int)blockIdx.x * 64 + lane;
  float sb = 0.f, sg = 0.f;
  if (c < a.channels) {
#pragma unroll 4
    for (int i = wave; i < parts; i += 16) {
      const float* q = a.part + (size_t)i * 2 * a.channels + c;
      sb += q[0];
      sg += q[a.channels];
    }
  }
  red[wave][0][lane] = sb;
  red[wave][1][lane] = sg;
  __syncthreads();
  if (wave < 2 && c < a.channels) {
    float t = 0.f;
    for (int w = 0; w < 16; w++) t += red[w][wave][lane];
    float* out = wave ? a.dgamma : a.dbeta;
    if (out) out[c] = t;
  }
}

// How a call runs. groups 0: by rows (channels fewer than a column's, or groups wider than a workgroup joins); else on slabs of
// that many groups, `threads` threads a workgroup with up to `each` points each, the row's points in `splits` shares: 1 where a
// batch row's slab fits the registers of 1024 threads with 8 points each (128 KB of 16-bit values). A slab is the fewest groups
// that give four whole columns where such fit.
struct SlabShape {
  int groups = 0, threads = 0, each = 0, splits = 1;
};
SlabShape slab_shape(int points, int groups, int width, int vec, int batch) {
  SlabShape best;
  if (points < 1 || width < 1) return best;
  for (int sg = 1; sg <= groups; sg++) {
    if (groups % sg || sg * width < vec) continue;
    const int w = sg * width, cols = (w + vec - 1) / vec;
    if (w > 1024) break;
    const int lanes = 1024 / cols, each = (points + lanes - 1) / lanes;
    if (each > 8) break;
    // As few points a thread as 1024 threads allow, and no more threads than those take (361 points of 6 columns: 3 points and
    // 768 threads, where 1024 threads left a third of the work to empty points).
    best = {sg, std::max(round_up((points + each - 1) / each * cols, 64), round_up(w, 64)), each, 1};
    if (w >= 4 * vec) break;
  }
  // Where there are more workgroups than CUs, four points a thread rather than one or two: smaller workgroups, more of them at once
  // on a CU. 143 x 194 points of 864 bf16 channels in 24 groups 110 -> 28 us and backward 108 -> 33; 512 boards of 361 x 128 f32 in 8
  // groups 59 -> 40 and 78 -> 57. (Three points stay, for both directions: 128 boards of 361 x 384 bf16 with mish backward 45 us, 59 with
  // four; forward with four is not measured.)
  if (best.groups && best.each < 3 && (long long)batch * (groups / best.groups) > kCUs) {
    const int w = best.groups * width, cols = (w + vec - 1) / vec;
    best.each = std::min(4, points);
    best.threads = std::max(round_up((points + best.each - 1) / best.each * cols, 64), round_up(w, 64));
  }
  if (best.groups) return best;
  for (int sg = 1; sg <= groups; sg++) {
    if (groups % sg || sg * width < vec) continue;
    const int w = sg * width, cols = (w + vec - 1) / vec;
    if (w > 1024) break;
    // (Two workgroups of 512 threads a CU; the joins take a thread a channel.)
    const int threads = w > 512 ? 1024 : 512, share = threads / cols * 8;
    best = {sg, threads, 8, (points + share - 1) / share};
    if (w >= 4 * vec) break;
  }
  return best;
}
// The same for a call: byte offsets within a share have 31 bits.
SlabShape slab_shape(const NormArgs& n, int size) {
  const SlabShape f = slab_shape(n.points, n.groups, n.width, 16 / size, n.batch);
  const long long ld = std::max(std::max(n.ldx, n.ldy), std::max(n.lddy, n.lddx));
  const long long share = f.splits == 1 ? n.points : 8 * 1024;
  return share * ld < (1ll << 31) / size ? f : SlabShape();
}

NormArgs norm_args(const kg_group_norm_args& a) {
  NormArgs n = {};
  n.x = a.x; n.ldx = a.ldx;
  n.y = a.y; n.ldy = a.ldy;
  n.dy = a.dy; n.lddy = a.lddy;
  n.dx = a.dx; n.lddx = a.lddx;
  n.mask = a.mask; n.gamma = a.gamma; n.beta = a.beta;
  n.mean = a.mean; n.rstd = a.rstd;
  n.dgamma = a.dgamma; n.dbeta = a.dbeta;
  n.batch = a.batch; n.points = a.points; n.channels = a.channels; n.groups = a.groups;
  n.width = a.channels / a.groups;
  n.splits = group_norm_splits(a.batch, a.points, a.channels);
  n.past = (long long)a.batch * a.points * a.channels * (a.type == KG_PRECISION_F32 ? 4 : 2) > kPastBytes;
  n.eps = (float)a.eps;
  n.part = (float*)a.workspace;
  return n;
}

template <typename T, int ACT>
void norm_forward_act(NormArgs& n, hipStream_t s) {
  const SlabShape f = slab_shape(n, sizeof(T));
  if (!f.groups) {
    const dim3 grid(n.batch * n.splits);
    launch_k(norm_stats_kernel<T>, grid, GT, 0, s, n);
    launch_k(norm_apply_kernel<T, ACT>, grid, GT, 0, s, n);
    return;
  }
  n.slab_groups = f.groups;
  n.each = f.each;
  n.splits = f.splits;
  const dim3 grid((n.batch * f.splits * (n.groups / f.groups) + 7) / 8 * 8);
  const size_t lds = slab_lds_bytes(kVec<T>, f.threads, (f.groups * n.width + kVec<T> - 1) / kVec<T>, f.groups, false);
  if (f.splits > 1) {
    launch_k(norm_slab_kernel<T, ACT_ID, 1024, 8, true>, grid, f.threads, lds, s, n);
    launch_k(norm_slab_apply_kernel<T, ACT, 1024, 8>, grid, f.threads, lds, s, n);
  } else if (f.each <= 4) launch_k(norm_slab_kernel<T, ACT, 1024, 4, false>, grid, f.threads, lds, s, n);
  else launch_k(norm_slab_kernel<T, ACT, 1024, 8, false>, grid, f.threads, lds, s, n);
}

template <typename T>
void norm_forward(NormArgs& n, int act, hipStream_t s) {
  switch (act) {
    case ACT_RELU: norm_forward_act<T, ACT_RELU>(n, s); break;
    case ACT_MISH: norm_forward_act<T, ACT_MISH>(n, s); break;
    case ACT_SILU: norm_forward_act<T, ACT_SILU>(n, s); break;
    default: norm_forward_act<T, ACT_ID>(n, s); break;
  }
}

template <typename T, int ACT>
void norm_backward_act(NormArgs& n, hipStream_t s) {
  const SlabShape f = slab_shape(n, sizeof(T));
  const dim3 columns((n.channels + 63) / 64), join((n.batch * n.groups + GT / 64 - 1) / (GT / 64));
  if (f.groups) {
    n.slab_groups = f.groups;
    n.each = f.each;
    n.splits = f.splits;
  }
  // part [batch][splits][2][channels], counts [batch][splits], sums [batch][splits][2][groups], means [batch][2][groups]
  const size_t parts = (size_t)n.batch * n.splits;
  n.counts = n.part + parts * 2 * n.channels;
  n.sums = n.counts + parts;
  n.means = n.sums + parts * 2 * n.groups;
  if (n.batch && !f.groups) {
    const dim3 grid(n.batch * n.splits);
    launch_k(norm_back_sums_kernel<T, ACT>, grid, GT, 0, s, n);
    launch_k(norm_back_join_kernel, join, GT, 0, s, n);
    launch_k(norm_back_apply_kernel<T, ACT>, grid, GT, 0, s, n);
  } else if (n.batch) {
    const dim3 grid((n.batch * f.splits * (n.groups / f.groups) + 7) / 8 * 8);
    const size_t lds = slab_lds_bytes(kVec<T>, f.threads, (f.groups * n.width + kVec<T> - 1) / kVec<T>, f.groups, true);
    if (f.splits > 1) {
      launch_k(norm_back_slab_kernel<T, ACT, 1024, 8, true, false>, grid, f.threads, lds, s, n);
      launch_k(norm_back_slab_apply_kernel<T, ACT, 1024, 8>, grid, f.threads, lds, s, n);
    } else if (f.each > 4) launch_k(norm_back_slab_kernel<T, ACT, 1024, 8, false, false>, grid, f.threads, lds, s, n);
    else if (grid.x <= kCUs) launch_k(norm_back_slab_kernel<T, ACT, 1024, 4, false, true>, grid, f.threads, lds, s, n);
    else launch_k(norm_back_slab_kernel<T, ACT, 1024, 4, false, false>, grid, f.threads, lds, s, n);
  }
  if (n.dgamma || n.dbeta) launch_k(norm_back_params_kernel, columns, 1024, 0, s, n, n.batch * n.splits);
}

template <typename T>
void norm_backward(NormArgs& n, int act, hipStream_t s) {
  switch (act) {
    case ACT_RELU: norm_backward_act<T, ACT_RELU>(n, s); break;
    case ACT_MISH: norm_backward_act<T, ACT_MISH>(n, s); break;
    case ACT_SILU: norm_backward_act<T, ACT_SILU>(n, s); break;
    default: norm_backward_act<T, ACT_ID>(n, s); break;
  }
}

}  // namespace

int group_norm_splits(int batch, int points, int channels) {
  // (A row of fewer channels takes a thread all the same: 36 x 11761 points of one channel took 53 us forward and 96
  // backward by its elements alone, 16 and 38 so.)
  const long long want = ((long long)points * std::max(channels, 8) + kSplitTarget - 1) / kSplitTarget;
  const long long most = batch > 0 ? (2048 + batch - 1) / batch : 1;
  long long n = want < most ? want : most;
  if (n > points) n = points;
  return n < 1 ? 1 : (int)n;
}

// For any type and strides: the most shares that one of the ways to run it takes.
size_t group_norm_workspace(int batch, int points, int channels, int groups, bool backward) {
  int splits = group_norm_splits(batch, points, channels);
  for (int vec = 4; vec <= 8; vec += 4) splits = std::max(splits, slab_shape(points, groups, channels / groups, vec, batch).splits);
  const size_t parts = (size_t)batch * splits;
  const size_t floats = parts * (backward ? 2 * ((size_t)channels + groups) + 1 : 3 * (size_t)groups) + (backward ? (size_t)batch * 2 * groups : 0);
  return (floats * 4 + 255) / 256 * 256;
}

bool group_norm_fits(const kg_group_norm_args& a) {
  const NormArgs n = norm_args(a);
  const SlabShape f = slab_shape(n, a.type == KG_PRECISION_F32 ? 4 : 2);
  const long long workgroups = f.groups ? (long long)n.batch * f.splits * (n.groups / f.groups) + 7 : (long long)n.batch * n.splits,
                  joins = ((long long)n.batch * n.groups + GT / 64 - 1) / (GT / 64);
  return std::max(workgroups * (f.groups ? f.threads : GT), joins * GT) < 1ll << 32;
}

void launch_group_norm(const kg_group_norm_args& a, hipStream_t s) {
  NormArgs n = norm_args(a);
  switch (a.type) {
    case PREC_F32: norm_forward<float>(n, a.act, s); break;
    case PREC_F16: norm_forward<f16>(n, a.act, s); break;
    default: norm_forward<bf16>(n, a.act, s); break;
  }
  KGX_CHECK_LAUNCH();
}

void launch_group_norm_backward(const kg_group_norm_args& a, hipStream_t s) {
  NormArgs n = norm_args(a);
  switch (a.type) {
    case PREC_F32: norm_backward<float>(n, a.act, s); break;
    case PREC_F16: norm_backward<f16>(n, a.act, s); break;
    default: norm_backward<bf16>(n, a.act, s); break;
  }
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
