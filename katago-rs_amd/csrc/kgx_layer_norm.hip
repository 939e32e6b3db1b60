// Layer norm and RMS norm over the channels of a row, forward and backward (kg_layer_norm, kg_layer_norm_backward).
//
// With h = (x - mean) rstd: y = h gamma + beta; backward, with d = dy gamma, dx = rstd (d - mean(d) - h mean(d h)) over the
// row's channels, dgamma = sum of dy h and dbeta = sum of dy over the rows. RMS norm has no mean, in either direction.
//
// The variance comes from the deviations d from the mean as a float sum gives it. Where that mean is far from 0, their own mean says
// what its rounding left, and is taken out of both (correction).
#include <algorithm>

#include "kgx_device.h"
#include "kgx_learn.h"
#include "kgx_rows.h"

namespace kgx {

namespace {

constexpr int LT = 256;        // threads of a workgroup
constexpr int kMostParts = 512;  // of the rows, for the sums over them

struct LayerArgs {
  const void *x, *dy;
  void *y, *dx;
  long long ldx, ldy, lddy, lddx;
  const float *gamma, *beta;
  float *mean, *rstd, *dgamma, *dbeta;
  float* parts;  // [parts][2][channels] sums of dy h and dy over a part's rows
  int rows, channels, rms, split;
  double eps;
};

// (NaN stays NaN: a comparison, not fmax.)
__device__ __forceinline__ float root_of(double variance, double eps) { return (float)(1.0 / sqrt((variance < 0.0 ? 0.0 : variance) + eps)); }

// The deviations' mean where it says something of the row's mean. Below 2^-22 of their size it is their own rounding: values on a
// coarse grid less a mean off that grid are rounded the same way all over a binade (2047 rows of 10007 f16 whose mean was 0.01 of
// their size: the means were off by 4e-6 with it, by 8e-8 without).
__device__ __forceinline__ double correction(double off, double square, int channels) {
  const double m = off / channels, size = square / channels;
  return m * m > 0x1p-44 * size ? m : 0.0;
}

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
      for (int c = tid; c < a.channels; c += LT) sum += (float)x[c];
      mean = (float)(row_sum<LT>(sum, red) / a.channels);
    }
    float off = 0.f, square = 0.f;
    for (int c = tid; c < a.channels; c += LT) {
      const float d = (float)x[c] - mean;
      off += d;
      square = __builtin_fmaf(d, d, square);
    }
    const double squares = row_sum<LT>(square, red);
    const double m = a.rms ? 0.0 : correction(row_sum<LT>(off, red), squares, a.channels);
    const float rstd = root_of(squares / a.channels - m * m, a.eps), shift = (float)m;
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

template <typename T>
__global__ __launch_bounds__(LT) void layer_norm_back_kernel(LayerArgs a) {
  __shared__ float red[16];
  const int tid = threadIdx.x;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + (size_t)row * a.ldx;
    const T* dy = (const T*)a.dy + (size_t)row * a.lddy;
    T* dx = (T*)a.dx + (size_t)row * a.lddx;
    const float mean = a.rms ? 0.f : a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int c = tid; c < a.channels; c += LT) {
      const float d = (float)dy[c] * (a.gamma ? a.gamma[c] : 1.f);
      s1 += d;
      s2 = __builtin_fmaf(d, ((float)x[c] - mean) * rstd, s2);
    }
    const float m1 = a.rms ? 0.f : (float)(row_sum<LT>(s1, red) / a.channels), m2 = (float)(row_sum<LT>(s2, red) / a.channels);
    for (int c = tid; c < a.channels; c += LT) {
      const float d = (float)dy[c] * (a.gamma ? a.gamma[c] : 1.f), h = ((float)x[c] - mean) * rstd;
      dx[c] = to_t<T>(rstd * __builtin_fmaf(-h, m2, d - m1));
    }
  }
}

// The sums over a part of the rows, a thread a channel.
template <typename T>
__global__ __launch_bounds__(LT) void layer_norm_sums_kernel(LayerArgs a) {
  const int per = (a.rows + a.split - 1) / a.split, part = blockIdx.y, first = part * per, last = min(first + per, a.rows);
  for (int c = blockIdx.x * LT + threadIdx.x; c < a.channels; c += gridDim.x * LT) {
    float s1 = 0.f, s2 = 0.f;
    for (int row = first; row < last; row++) {
      const float d = (float)((const T*)a.dy)[(size_t)row * a.lddy + c];
      const float h = ((float)((const T*)a.x)[(size_t)row * a.ldx + c] - (a.rms ? 0.f : a.mean[row])) * a.rstd[row];
      s1 = __builtin_fmaf(d, h, s1);
      s2 += d;
    }
    a.parts[(size_t)part * 2 * a.channels + c] = s1;
    a.parts[((size_t)part * 2 + 1) * a.channels + c] = s2;
  }
}

// The parts' sums joined in double.
__global__ __launch_bounds__(LT) void layer_norm_params_kernel(LayerArgs a) {
  for (long long i = (long long)blockIdx.x * LT + threadIdx.x; i < 2ll * a.channels; i += (long long)gridDim.x * LT) {
    double s = 0.0;
    for (int p = 0; p < a.split; p++) s += (double)a.parts[(size_t)p * 2 * a.channels + i];
    float* out = i < a.channels ? a.dgamma : a.dbeta;
    if (out) out[i < a.channels ? i : i - a.channels] = (float)s;
  }
}

int parts_of(int rows) { return std::min(std::max(rows / 8, 1), kMostParts); }

LayerArgs args_of(const kg_layer_norm_args& a) {
  LayerArgs p;
  p.x = a.x; p.ldx = a.ldx;
  p.y = a.y; p.ldy = a.ldy;
  p.dy = a.dy; p.lddy = a.lddy;
  p.dx = a.dx; p.lddx = a.lddx;
  p.gamma = a.gamma; p.beta = a.beta;
  p.mean = a.mean; p.rstd = a.rstd;
  p.dgamma = a.dgamma; p.dbeta = a.dbeta;
  p.parts = (float*)a.workspace;
  p.rows = a.rows; p.channels = a.channels; p.rms = a.rms != 0;
  p.split = parts_of(a.rows);
  p.eps = a.eps;
  return p;
}

template <typename T>
void backward_typed(const LayerArgs& p, hipStream_t s) {
  launch_k(layer_norm_back_kernel<T>, dim3(row_grid(p.rows, 1)), LT, 0, s, p);
  if (p.dgamma || p.dbeta)
    launch_k(layer_norm_sums_kernel<T>, dim3(std::min((p.channels + LT - 1) / LT, 1024), p.split), LT, 0, s, p);
}

}  // namespace

size_t layer_norm_workspace(int rows, int channels) {
  if (rows < 1 || channels < 1) return 0;
  return (size_t)parts_of(rows) * 2 * channels * sizeof(float);
}

void launch_layer_norm(const kg_layer_norm_args& a, hipStream_t s) {
  const LayerArgs p = args_of(a);
  const dim3 grid(row_grid(p.rows, 1));
  switch (a.type) {
    case PREC_F32: launch_k(layer_norm_kernel<float>, grid, LT, 0, s, p); break;
    case PREC_F16: launch_k(layer_norm_kernel<f16>, grid, LT, 0, s, p); break;
    default: launch_k(layer_norm_kernel<bf16>, grid, LT, 0, s, p); break;
  }
  KGX_CHECK_LAUNCH();
}

void launch_layer_norm_backward(const kg_layer_norm_args& a, hipStream_t s) {
  LayerArgs p = args_of(a);
  if (!p.rows) p.split = 0;  // (the sums over no rows are 0)
  else switch (a.type) {
    case PREC_F32: backward_typed<float>(p, s); break;
    case PREC_F16: backward_typed<f16>(p, s); break;
    default: backward_typed<bf16>(p, s); break;
  }
  if (p.dgamma || p.dbeta) launch_k(layer_norm_params_kernel, dim3((int)std::min((2ll * p.channels + LT - 1) / LT, 65536ll)), LT, 0, s, p);
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
