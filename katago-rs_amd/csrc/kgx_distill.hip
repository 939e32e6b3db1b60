// The distillation loss from a teacher's top logits, with its gradient (kg_distill_loss).
//
// The teacher's q is known on a row's listed columns alone, so the other columns share one gradient factor: with p = softmax(s z)
// and m the mass that q has, grad_j = w s (m p_j - q_j) where listed, else w s p_j (m - rest / R), R = the others' p. The
// listed columns are a few dozen values: they are read apart and go into double, and the row's pass over its columns sums the
// others alone, relative to their own maximum. (Sums of both would leave R, and m - rest / R, to a cancellation.)
//
// A listed column is found by its chunk of 16 bytes: lists hang from one head for each chunk that a workgroup holds at a time, so a
// thread asks for its own chunks' lists and nobody searches. Columns that are listed twice meet in one list, where the first counts.
#include <algorithm>
#include <climits>

#include "kgx_device.h"
#include "kgx_learn.h"
#include "kgx_rows.h"

namespace kgx {

namespace {

struct DistillRows {
  const void* logits;
  const unsigned char* legal;
  void* grad;
  const int* index;
  const void* top;
  long long ld, ld_legal, ld_grad, ld_index, ld_top;
  const float *lse, *weight;
  float* loss;
  int rows, columns, k, top_type, past;
  double scale;
};

// A row's listed columns in LDS: the lists (link: column, or -1 where it does not count, and 1 + the next entry; heads: 1 + the
// first), the student's logits and the teacher's; later z holds the entries' gradients.
struct Listed {
  int* heads;
  int2* link;
  float *z, *t;
  int k;
  __device__ __forceinline__ Listed(char* lds, int slots, int k_) : k(k_) {
    link = (int2*)lds;
    z = (float*)(link + k);
    t = z + k;
    heads = (int*)(t + k);
  }
  static size_t bytes(int slots, int k) { return (size_t)k * 16 + (size_t)slots * 4; }
};

// LDS written before is read after: a wave's accesses are in order by themselves.
template <int NT>
__device__ __forceinline__ void row_sync() {
  if constexpr (NT == 64) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  } else {
    lds_barrier();
  }
}

__device__ __forceinline__ float top_value(const DistillRows& a, int row, int i) {
  const size_t at = (size_t)row * a.ld_top + i;
  switch (a.top_type) {
    case PREC_F32: return ((const float*)a.top)[at];
    case PREC_F16: return (float)((const f16*)a.top)[at];
    default: return (float)((const bf16*)a.top)[at];
  }
}

// Fills the lists of a row; slot: a column's head.
template <typename T, int NT, int SLOTS, typename Slot>
__device__ __forceinline__ void list_row(const DistillRows& a, int row, const T* z, const unsigned char* legal, const Listed& l,
                                         const Slot& slot) {
  const int tid = threadIdx.x % NT;
#pragma unroll
  for (int i = 0; i < SLOTS / NT; i++) l.heads[tid + i * NT] = 0;
  row_sync<NT>();
  for (int i = tid; i < l.k; i += NT) {
    int c = a.index[(size_t)row * a.ld_index + i], next = 0;
    if ((unsigned)c >= (unsigned)a.columns || (legal && !legal[c])) c = -1;
    const float t = top_value(a, row, i);
    if (c >= 0) next = atomicExch(&l.heads[slot(c)], i + 1);
    l.link[i] = int2{c, next};
    l.z[i] = c >= 0 ? (float)z[c] : -INFINITY;
    l.t[i] = c >= 0 ? t : -INFINITY;
  }
  row_sync<NT>();
  // Of entries that name one column the first counts.
  unsigned gone = 0;
  for (int i = tid, b = 0; i < l.k; i += NT, b++) {
    const int c = l.link[i].x;
    if (c < 0) continue;
    for (int h = l.heads[slot(c)]; h; h = l.link[h - 1].y)
      if (h - 1 < i && l.link[h - 1].x == c) gone |= 1u << b;
  }
  row_sync<NT>();
  for (int i = tid, b = 0; i < l.k; i += NT, b++)
    if (gone >> b & 1) {
      l.link[i].x = -1;
      l.z[i] = l.t[i] = -INFINITY;
    }
  row_sync<NT>();
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// What the others' gradient takes: grad_j = each e^((z_j - top) s). part: the row takes part.
struct DistillFactors {
  float each;
  int part;
};

// The row's loss, the listed columns' gradients (into l.z) and the others' factor, from the others' maximum and their sum of
// e^((z - top) s), 0 where there are none. One wave computes it, in double: what is left of a loss between near distributions
// are differences of logarithms.
__device__ __forceinline__ DistillFactors distill_row(const DistillRows& a, int row, const Listed& l, float top, double total, bool writes) {
  const int lane = threadIdx.x & 63;
  const double s = a.scale, none = -(double)INFINITY;
  float z_max = -INFINITY, t_max = -INFINITY;
  bool any = false;
  for (int i = lane; i < l.k; i += 64) {
    z_max = fmaxf(z_max, l.z[i]);
    t_max = fmaxf(t_max, l.t[i]);
    any |= l.link[i].x >= 0;
  }
  any = __ballot(any) != 0;
  z_max = wave_reduce<true>(z_max);
  t_max = wave_reduce<true>(t_max);
  // (A sum that is NaN takes part, and makes everything NaN.)
  const bool others = !(total == 0.0);
  const double lo = others ? (double)top * s + log_sum(total) : none;
  double z_top = fmax((double)z_max * s, lo), t_top = (double)t_max * s;
  if (z_top == none) z_top = 0.0;
  if (t_top == none) t_top = 0.0;
  double z_sum = 0.0, t_sum = 0.0;
  for (int i = lane; i < l.k; i += 64) {
    z_sum += exp((double)l.z[i] * s - z_top);
    if (!a.lse) t_sum += exp((double)l.t[i] * s - t_top);
  }
  z_sum = wave_sum(z_sum) + (others ? exp(lo - z_top) : 0.0);
  t_sum = wave_sum(t_sum);
  const double lse = z_top + log_sum(z_sum);
  const double t_lse = a.lse ? (double)a.lse[row] : t_top + log_sum(t_sum);
  DistillFactors f = {0.f, any && !(z_sum == 0.0) && (a.lse || !(t_sum == 0.0))};
  double loss = 0.0, mass = 0.0;
  if (f.part) {
    for (int i = lane; i < l.k; i += 64) {
      const double x = (double)l.t[i] * s - t_lse, q = l.link[i].x < 0 ? 0.0 : exp(x);
      mass += q;
      loss += q == 0.0 ? 0.0 : q * (x - ((double)l.z[i] * s - lse));
    }
    mass = wave_sum(mass);
    loss = wave_sum(loss);
    double rest = 0.0;
    if (a.lse) {
      if (others && mass < 1.0) {
        rest = 1.0 - mass;
        loss += rest * (log_sum(rest) - (lo - lse));
      }
      mass += rest;
    } else {
      mass = 1.0 + 0.0 * t_lse;  // (a NaN among the teacher's is everyone's)
    }
    const double w = a.weight ? (double)a.weight[row] : 1.0, ws = w * s;
    loss *= w;
    if (others) f.each = (float)(ws * (mass * exp(lo - lse) - rest) / total);
    for (int i = lane; i < l.k; i += 64) {
      const double x = (double)l.t[i] * s - t_lse, q = l.link[i].x < 0 ? 0.0 : exp(x);
      l.z[i] = (float)(ws * (mass * exp((double)l.z[i] * s - lse) - q));
    }
  }
  if (writes) a.loss[row] = (float)loss;
  return f;
}

// Rows shorter than 16 bytes: a wave a row, a lane a column.
template <typename T>
__global__ __launch_bounds__(64) void distill_short_kernel(DistillRows a) {
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x;
  const Listed l(lds, 64, a.k);
  const Base2 c2(a.scale);
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const unsigned char* legal = a.legal ? a.legal + (size_t)row * a.ld_legal : nullptr;
    row_sync<64>();  // (the last row's lists have been read)
    list_row<T, 64, 64>(a, row, z, legal, l, [](int c) { return c; });
    int mine = -1;  // the entry that lists this lane's column
    for (int h = l.heads[lane]; h; h = l.link[h - 1].y)
      if (l.link[h - 1].x >= 0) mine = h - 1;
    const bool in = lane < a.columns && (!legal || legal[lane]) && mine < 0;
    const float v = in ? (float)z[lane] : -INFINITY;
    float top = wave_reduce<true>(v);
    const float e = exp_of(v - (top == -INFINITY ? 0.f : top), c2);
    const float sum = wave_reduce<false>(e);
    const DistillFactors f = distill_row(a, row, l, top, (double)sum, lane == 0);
    row_sync<64>();
    if (a.grad && lane < a.columns)
      ((T*)a.grad)[(size_t)row * a.ld_grad + lane] = to_t<T>(!f.part ? 0.f : mine >= 0 ? l.z[mine] : in ? e * f.each : 0.f);
  }
}

// -infinity in the place of listed columns, of the E chunks of a thread from chunk c0 on.
template <typename T, int NT, int E>
__device__ __forceinline__ void remove_listed(const Listed& l, int tid, const Chunks<T>& at, u32x4 (&raw)[E], int c0) {
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (at.none(c0 + e * NT)) break;
    const int c = tid + c0 + e * NT;
    for (int h = l.heads[tid + e * NT]; h; ) {
      const int2 entry = l.link[h - 1];
      if (entry.x >= 0 && at.of(entry.x) == c) {
        const int j0 = entry.x - at.start(c);
#pragma unroll
        for (int j = 0; j < kVec<T>; j++) remove<T>(raw[e], j, j == j0);
      }
      h = entry.y;
    }
  }
}

// Any row of at least 16 bytes: E chunks of each thread at a time relative to the running maximum, and again for the gradient.
template <typename T, int NT, int E>
__global__ __launch_bounds__(NT) void distill_long_kernel(DistillRows a) {
  constexpr int V = kVec<T>, SLOTS = NT * E;
  extern __shared__ __align__(16) char lds[];
  __shared__ float red[16];
  __shared__ DistillFactors box;
  const int tid = threadIdx.x;
  const Listed l(lds, SLOTS, a.k);
  const Base2 c2(a.scale);
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const unsigned char* legal = a.legal ? a.legal + (size_t)row * a.ld_legal : nullptr;
    T* g = a.grad ? (T*)a.grad + (size_t)row * a.ld_grad : nullptr;
    const Chunks<T> at(a.columns, g ? g : z);
    lds_barrier();  // (the last row's lists and factors have been read)
    list_row<T, NT, SLOTS>(a, row, z, legal, l, [&](int c) { return at.of(c) % SLOTS; });
    auto piece = [&](int c0, u32x4(&raw)[E]) {
      u32x4 unused[1];
      load_row<T, NT, E>(z, tid, at, raw, c0);
      if (legal) remove_illegal<T, NT, E, false>(legal, tid, at, raw, unused, c0);
      remove_past<T, NT, E>(tid, at, raw, c0);
    };
    Running run;
    for (int c0 = 0; !at.none(c0); c0 += NT * E) {
      u32x4 raw[E];
      piece(c0, raw);
      remove_listed<T, NT, E>(l, tid, at, raw, c0);
      float f[E * V];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const bool in = !at.none(c0 + e * NT);
#pragma unroll
        for (int j = 0; j < V; j++) f[e * V + j] = in ? element<T>(raw[e], j) : -INFINITY;
      }
      run.add<E * V>(f, c2);
    }
    float moved;
    run.join<NT>(c2, red, moved);
    if (tid < 64) {
      const DistillFactors mine = distill_row(a, row, l, run.top, run.total, tid == 0);
      if (tid == 0) box = mine;
    }
    lds_barrier();
    if (!g) continue;
    const DistillFactors f = box;
    const bool part = __builtin_amdgcn_readfirstlane(f.part);
    const float top = run.top == -INFINITY ? 0.f : run.top;
    for (int c0 = 0; !at.none(c0); c0 += NT * E) {
      u32x4 raw[E];
      if (part) piece(c0, raw);
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (at.none(c0 + e * NT)) break;
        const int c = tid + c0 + e * NT;
        float gf[V] = {};
        if (part) {
          // (A column without mass has no gradient, whatever the factor. A listed one's place is filled below.)
#pragma unroll
          for (int j = 0; j < V; j++) {
            const float ex = __builtin_amdgcn_exp2f((element<T>(raw[e], j) - top) * c2.hi);
            gf[j] = ex == 0.f ? 0.f : ex * f.each;
          }
          for (int h = l.heads[tid + e * NT]; h; ) {
            const int2 entry = l.link[h - 1];
            if (entry.x >= 0 && at.of(entry.x) == c) {
              const int j0 = entry.x - at.start(c);
#pragma unroll
              for (int j = 0; j < V; j++) gf[j] = j == j0 ? l.z[h - 1] : gf[j];
            }
            h = entry.y;
          }
        }
        store_gradient<T>(g, c, at.whole(c0 + e * NT, NT), a.past, at, gf);
      }
    }
  }
}

template <typename T>
void distill_typed(const DistillRows& p, hipStream_t s) {
  const dim3 groups(row_grid(p.rows, 1));
  if (p.columns < kVec<T>) launch_k(distill_short_kernel<T>, groups, 64, Listed::bytes(64, p.k), s, p);
  else launch_k(distill_long_kernel<T, 256, 4>, groups, 256, Listed::bytes(1024, p.k), s, p);
}

}  // namespace

size_t distill_loss_workspace(int rows, int columns) { return 0; }

void launch_distill_loss(const kg_distill_loss_args& a, hipStream_t s) {
  DistillRows p;
  p.logits = a.logits; p.ld = a.ld;
  p.legal = a.legal; p.ld_legal = a.ld_legal;
  p.grad = a.grad; p.ld_grad = a.ld_grad;
  p.index = a.top_index; p.ld_index = a.ld_index;
  p.top = a.top_logits; p.ld_top = a.ld_top;
  p.lse = a.teacher_lse; p.weight = a.weight;
  p.loss = a.loss;
  p.rows = a.rows; p.columns = a.columns; p.k = a.k; p.top_type = a.top_type;
  p.past = gradient_past(a.rows, a.columns, a.type);
  p.scale = a.logit_scale;
  switch (a.type) {
    case PREC_F32: distill_typed<float>(p, s); break;
    case PREC_F16: distill_typed<f16>(p, s); break;
    default: distill_typed<bf16>(p, s); break;
  }
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
