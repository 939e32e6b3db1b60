// Group norm with an activation on channels-last rows under the board mask, forward and backward (kg_group_norm,
// kg_group_norm_backward).
//
// Bound by memory. A workgroup takes a share of one batch row's points with all their channels, so that every access runs
// along whole rows however wide or odd the groups are; a thread keeps its column of 16 bytes for all its points, with the
// channels' parameters in registers. The statistics of a group cross workgroups, so each direction is a reduction launch
// and an elementwise one; the second reading of the same rows comes from the caches where they fit.
#include "kgx_device.h"
#include "kgx_learn.h"

namespace kgx {

namespace {

constexpr int GT = 256;         // threads of a workgroup
constexpr int kSplitTarget = 16384;  // elements a workgroup, about
constexpr int kMaxGroups = 2048;     // group statistics in LDS

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
template <typename T> constexpr int kVec = 16 / sizeof(T);
template <typename T> struct RowVec { typedef u16x8_any type; };
template <> struct RowVec<float> { typedef f32x4_any type; };

template <typename T>
__device__ __forceinline__ void load_vec(const T* p, int left, float (&f)[kVec<T>]) {
  if (left >= kVec<T>) {
    const typename RowVec<T>::type v = *(const typename RowVec<T>::type*)p;
#pragma unroll
    for (int j = 0; j < kVec<T>; j++) {
      if constexpr (std::is_same<T, float>::value) f[j] = v[j];
      else if constexpr (std::is_same<T, bf16>::value) f[j] = __uint_as_float((unsigned)v[j] << 16);
      else f[j] = (float)__builtin_bit_cast(f16, (unsigned short)v[j]);
    }
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
  float* sums;     // backward: [batch][2][groups]
  int batch, points, channels, groups, width, splits;  // width: channels of a group
  float eps;
};

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
// sums each of its channels relative to the first value that it meets (no cancellation for a mean far from 0); the
// parts are joined pairwise exactly: M2 = sum M2_i + n_i (mean_i - mean)^2.
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
    float pivot[V], s1[V], s2[V], n = 0.f;
#pragma unroll
    for (int j = 0; j < V; j++) pivot[j] = s1[j] = s2[j] = 0.f;
    if (w.lane < w.lanes) {
      const T* x = (const T*)a.x + (size_t)b * a.points * a.ldx + c0;
      for (int p = p0 + w.lane; p < p1; p += w.lanes) {
        if (a.mask && a.mask[(size_t)b * a.points + p] == 0.f) continue;
        float f[V];
        load_vec<T>(x + (size_t)p * a.ldx, left, f);
        if (n == 0.f) {
#pragma unroll
          for (int j = 0; j < V; j++) pivot[j] = f[j];
        }
        n += 1.f;
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float d = f[j] - pivot[j];
          s1[j] += d;
          s2[j] = __builtin_fmaf(d, d, s2[j]);
        }
      }
    }
    const float inv = n > 0.f ? 1.f / n : 0.f;
    s_n[tid] = n;
#pragma unroll
    for (int j = 0; j < V; j++) {
      const float mean = s1[j] * inv;
      s_mean[j * GT + tid] = pivot[j] + mean;
      s_m2[j * GT + tid] = fmaxf(__builtin_fmaf(-s1[j], mean, s2[j]), 0.f);
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
  for (int g = tid; g < a.groups; g += GT) {
    const float* in = a.part + (size_t)b * a.splits * 3 * a.groups + g;
    float n = 0.f, s = 0.f, m2 = 0.f;
    for (int i = 0; i < a.splits; i++) {
      const float* q = in + (size_t)i * 3 * a.groups;
      n += q[0];
      s = __builtin_fmaf(q[0], q[a.groups], s);
    }
    const float mean = n > 0.f ? s / n : 0.f;
    for (int i = 0; i < a.splits; i++) {
      const float* q = in + (size_t)i * 3 * a.groups;
      const float d = q[a.groups] - mean;
      m2 += q[2 * a.groups] + (q[0] > 0.f ? q[0] * d * d : 0.f);
    }
    const float rstd = 1.f / sqrtf((n > 0.f ? m2 / n : 0.f) + a.eps);
    g_mean[g] = mean;
    g_rstd[g] = rstd;
    if (k == 0) {
      a.mean[(size_t)b * a.groups + g] = mean;
      a.rstd[(size_t)b * a.groups + g] = rstd;
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
        for (int j = 0; j < V; j++) f[j] = act_f<ACT>(__builtin_fmaf(f[j] - mean[j], mul[j], add[j]));
      }
      store_vec<T>(y + (size_t)p * a.ldy, left, f);
    }
  }
}

// d act(a) / d a. Mish: with e = exp(a) and n = e (e + 2), tanh(softplus) = n / (n + 2) and 1 - tanh^2 = 4 (e + 1)^2 /
// (n + 2)^2, so the derivative n / (n + 2) + 4 a e (e + 1) / (n + 2)^2 has no cancellation but its own sign's.
template <int ACT>
__device__ __forceinline__ float act_slope(float v) {
  if constexpr (ACT == ACT_RELU) {
    return v > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == ACT_MISH) {
    const float e = __expf(fminf(v, 20.f)), n = e * (e + 2.f), r = __builtin_amdgcn_rcpf(n + 2.f);
    return v > 20.f ? 1.f : n * r + 4.f * v * (e * r) * ((e + 1.f) * r);
  } else if constexpr (ACT == ACT_SILU) {
    const float q = __builtin_amdgcn_rcpf(1.f + __expf(-v));
    return q * (1.f + v * (1.f - q));
  } else {
    return 1.f;
  }
}

// A column's parameters in the backward pass, and the gradient at the norm's output: da = dy act'(xh gamma + beta).
template <typename T, int ACT>
struct BackColumn {
  static constexpr int V = kVec<T>;
  float mean[V], rstd[V], gamma[V], beta[V];
  __device__ __forceinline__ void load(const NormArgs& a, int b, int c0) {
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int c = min(c0 + j, a.channels - 1), g = c / a.width;
      mean[j] = a.mean[(size_t)b * a.groups + g];
      rstd[j] = a.rstd[(size_t)b * a.groups + g];
      gamma[j] = a.gamma ? a.gamma[c] : 1.f;
      beta[j] = a.beta ? a.beta[c] : 0.f;
    }
  }
  __device__ __forceinline__ void grad(float x, float dy, int j, float& xh, float& da) const {
    xh = (x - mean[j]) * rstd[j];
    if constexpr (ACT == ACT_RELU && sizeof(T) == 4) {
      // The side of 0 in double: a float's rounding there would switch a whole gradient.
      const double v = __builtin_fma(((double)x - (double)mean[j]) * (double)rstd[j], (double)gamma[j], (double)beta[j]);
      da = v > 0.0 ? dy : 0.f;
    } else {
      da = dy * act_slope<ACT>(__builtin_fmaf(xh, gamma[j], beta[j]));
    }
  }
};

// Backward, first launch: sums of da and da xh over the workgroup's points, per channel.
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
          float xh, da;
          col.grad(f[j], d[j], j, xh, da);
          sb[j] += da;
          sg[j] = __builtin_fmaf(da, xh, sg[j]);
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
      out[a.channels + first * V + c] = tg;
    }
    if (first == 0 && tid == 0) {
      float t = 0.f;
      for (int l = 0; l < w.lanes; l++) t += s_n[l * w.cols];
      a.counts[blockIdx.x] = t;
    }
    __syncthreads();
  }
}

// Second launch. Workgroups [0, batch): a batch row's group sums, divided by the group's elements. The others: dgamma and
// dbeta of 64 channels each, four waves over the parts.
__global__ __launch_bounds__(GT) void norm_back_join_kernel(NormArgs a) {
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < a.batch) {
    const int b = blockIdx.x;
    float n = 0.f;
    for (int k = 0; k < a.splits; k++) n += a.counts[(size_t)b * a.splits + k];
    const float inv = n > 0.f ? 1.f / (n * (float)a.width) : 0.f;
    int share = 64;
    while (share > 1 && share * a.groups > GT) share >>= 1;
    const int sub = tid % share, per = GT / share;
    for (int gb = 0; gb < a.groups; gb += per) {
      const int g = gb + tid / share;
      float s1 = 0.f, s2 = 0.f;
      if (g < a.groups) {
        for (int i = sub; i < a.width * a.splits; i += share) {
          const int c = g * a.width + i % a.width, k = i / a.width;
          const float* q = a.part + ((size_t)b * a.splits + k) * 2 * a.channels + c;
          const float gm = a.gamma ? a.gamma[c] : 1.f;
          s1 = __builtin_fmaf(gm, q[0], s1);
          s2 = __builtin_fmaf(gm, q[a.channels], s2);
        }
      }
      for (int o = share >> 1; o >= 1; o >>= 1) { s1 += __shfl_xor(s1, o); s2 += __shfl_xor(s2, o); }
      if (g < a.groups && sub == 0) {
        a.sums[(size_t)b * 2 * a.groups + g] = s1 * inv;
        a.sums[(size_t)b * 2 * a.groups + a.groups + g] = s2 * inv;
      }
    }
  } else {
    __shared__ float red[4][2][64];
    const int c = ((int)blockIdx.x - a.batch) * 64 + (tid & 63), wave = tid >> 6, parts = a.batch * a.splits;
    float sb = 0.f, sg = 0.f;
    if (c < a.channels) {
      for (int i = wave; i < parts; i += 4) {
        const float* q = a.part + (size_t)i * 2 * a.channels + c;
        sb += q[0];
        sg += q[a.channels];
      }
    }
    red[wave][0][tid & 63] = sb;
    red[wave][1][tid & 63] = sg;
    __syncthreads();
    if (wave == 0 && c < a.channels) {
      if (a.dbeta) a.dbeta[c] = (red[0][0][tid] + red[1][0][tid]) + (red[2][0][tid] + red[3][0][tid]);
      if (a.dgamma) a.dgamma[c] = (red[0][1][tid] + red[1][1][tid]) + (red[2][1][tid] + red[3][1][tid]);
    }
  }
}

// Third launch: dx = rstd (da gamma - mean(da gamma) - xh mean(da gamma xh)).
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
    float m1[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int g = min(c0 + j, a.channels - 1) / a.width;
      m1[j] = a.sums[(size_t)b * 2 * a.groups + g];
      m2[j] = a.sums[(size_t)b * 2 * a.groups + a.groups + g];
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
          float xh, da;
          col.grad(f[j], d[j], j, xh, da);
          f[j] = col.rstd[j] * (da * col.gamma[j] - m1[j] - xh * m2[j]);
        }
      }
      store_vec<T>(dx + (size_t)p * a.lddx, left, f);
    }
  }
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
  n.eps = (float)a.eps;
  n.part = (float*)a.workspace;
  return n;
}

template <typename T>
void norm_forward(const NormArgs& n, int act, hipStream_t s) {
  const dim3 grid(n.batch * n.splits);
  launch_k(norm_stats_kernel<T>, grid, GT, 0, s, n);
  switch (act) {
    case ACT_RELU: launch_k(norm_apply_kernel<T, ACT_RELU>, grid, GT, 0, s, n); break;
    case ACT_MISH: launch_k(norm_apply_kernel<T, ACT_MISH>, grid, GT, 0, s, n); break;
    case ACT_SILU: launch_k(norm_apply_kernel<T, ACT_SILU>, grid, GT, 0, s, n); break;
    default: launch_k(norm_apply_kernel<T, ACT_ID>, grid, GT, 0, s, n); break;
  }
}

template <typename T, int ACT>
void norm_backward_act(const NormArgs& n, hipStream_t s) {
  const dim3 grid(n.batch * n.splits);
  if (n.batch) launch_k(norm_back_sums_kernel<T, ACT>, grid, GT, 0, s, n);
  launch_k(norm_back_join_kernel, dim3(n.batch + (n.channels + 63) / 64), GT, 0, s, n);
  if (n.batch) launch_k(norm_back_apply_kernel<T, ACT>, grid, GT, 0, s, n);
}

template <typename T>
void norm_backward(const NormArgs& n, int act, hipStream_t s) {
  switch (act) {
    case ACT_RELU: norm_backward_act<T, ACT_RELU>(n, s); break;
    case ACT_MISH: norm_backward_act<T, ACT_MISH>(n, s); break;
    case ACT_SILU: norm_backward_act<T, ACT_SILU>(n, s); break;
    default: norm_backward_act<T, ACT_ID>(n, s); break;
  }
}

}  // namespace

int group_norm_splits(int batch, int points, int channels) {
  const long long want = ((long long)points * channels + kSplitTarget - 1) / kSplitTarget;
  const long long most = batch > 0 ? (4096 + batch - 1) / batch : 1;
  long long n = want < most ? want : most;
  if (n > points) n = points;
  return n < 1 ? 1 : (int)n;
}

size_t group_norm_workspace(int batch, int points, int channels, int groups, bool backward) {
  const size_t parts = (size_t)batch * group_norm_splits(batch, points, channels);
  const size_t floats = backward ? parts * (2 * (size_t)channels + 1) + (size_t)batch * 2 * groups : parts * 3 * groups;
  return (floats * 4 + 255) / 256 * 256;
}

void launch_group_norm(const kg_group_norm_args& a, hipStream_t s) {
  const NormArgs n = norm_args(a);
  switch (a.type) {
    case PREC_F32: norm_forward<float>(n, a.act, s); break;
    case PREC_F16: norm_forward<f16>(n, a.act, s); break;
    default: norm_forward<bf16>(n, a.act, s); break;
  }
  KGX_CHECK_LAUNCH();
}

void launch_group_norm_backward(const kg_group_norm_args& a, hipStream_t s) {
  NormArgs n = norm_args(a);
  const size_t parts = (size_t)n.batch * n.splits;
  n.counts = n.part + parts * 2 * n.channels;
  n.sums = n.counts + parts;
  switch (a.type) {
    case PREC_F32: norm_backward<float>(n, a.act, s); break;
    case PREC_F16: norm_backward<f16>(n, a.act, s); break;
    default: norm_backward<bf16>(n, a.act, s); break;
  }
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
