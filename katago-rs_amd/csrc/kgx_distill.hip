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

struct Known;
struct Others {  // a row's columns that are not listed: their maximum, and the sum of e^((z - top) s)
  double total;
  float top;
};
struct DistillRows {
  const void* logits;
  const unsigned char* legal;
  void* grad;
  const int* index;
  const void* top;
  long long ld, ld_legal, ld_grad, ld_index, ld_top;
  const float *lse, *weight;
  float* loss;
  int rows, columns, k, top_type, past, list_bytes;  // list_bytes: of a wave's lists
  double scale;
  // Of rows that take a workgroup, by a launch before: what a wave knows of their entries (see Known).
  Known* known;
  Others *others, *parts;  // parts: of rows cut into `split` parts of `span` chunks
  int split, span, knowing;  // knowing: workgroups ahead of the parts', a wave of four for the entries of a row (0: by a launch before)
  double *share, *q;  // [rows][k]
  int* column;        // [rows][k], -1 where an entry does not count
};

// A row's listed columns in LDS: the lists (link: column, or -1 where it does not count, and 1 + the next entry, see also placed(); heads:
// 1 + the first), and the entries' gradients.
struct Lists {
  int* heads;
  int2* link;
  float* hot;
  int k;
  __device__ __forceinline__ Lists(char* lds, int k_) : k(k_) {
    link = (int2*)lds;
    hot = (float*)(link + k);
    heads = (int*)(hot + k);
  }
  static size_t bytes(int slots, int k) { return ((size_t)k * 12 + (size_t)slots * 4 + 15) / 16 * 16; }
};
// Those with what a wave learns of the entries: the student's share e^(s (z - their maximum)) and the teacher's q.
struct Listed : Lists {
  double *share, *q;
  __device__ __forceinline__ Listed(char* lds, int k_) : Lists(lds + (size_t)k_ * 16, k_) {
    share = (double*)lds;
    q = share + k;
  }
  static size_t bytes(int slots, int k) { return (size_t)k * 16 + Lists::bytes(slots, k); }
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

// A thread's entry of a row, asked for before the row itself: what is asked for later arrives later.
struct Entry {
  int c = -1;
  float t = -INFINITY;
  __device__ __forceinline__ Entry() {}
  __device__ __forceinline__ Entry(const DistillRows& a, int row, int i) {
    if (i < a.k) {
      c = a.index[(size_t)row * a.ld_index + i];
      t = top_value(a, row, i);
      if ((unsigned)c >= (unsigned)a.columns) c = -1;
    }
  }
};

// Fills the lists of a row, whose heads are 0, with NT threads; slot: a column's head; mine: this thread's first entry. The logits of
// both sides are left in share and q.
template <typename T, int NT, typename Slot>
__device__ __forceinline__ void list_row(const DistillRows& a, int row, const T* z, const unsigned char* legal, const Listed& l, const Entry& mine,
                                         const Slot& slot) {
  const int tid = threadIdx.x % NT;
  const auto entry = [&](int i) { return i < NT ? mine : Entry(a, row, i); };
#pragma unroll 1
  for (int i = tid; i < l.k; i += NT) {
    const int c = entry(i).c;
    l.link[i] = int2{c, c >= 0 ? atomicExch(&l.heads[slot(c)], i + 1) : 0};
  }
  row_sync<NT>();
  // Of entries that name one column the first counts. An illegal column's entries do not.
  unsigned gone = 0;
#pragma unroll 1
  for (int i = tid, b = 0; i < l.k; i += NT, b++) {
    const Entry own = entry(i);
    float v = -INFINITY;
    bool counts = own.c >= 0;
    if (counts) {
      v = (float)z[own.c];
      if (legal) counts = legal[own.c] != 0;
      for (int h = l.heads[slot(own.c)]; h; h = l.link[h - 1].y)
        if (h - 1 < i && l.link[h - 1].x == own.c) counts = false;
      if (!counts) gone |= 1u << b;
    }
    l.share[i] = (double)(counts ? v : -INFINITY);
    l.q[i] = (double)(counts ? own.t : -INFINITY);
  }
  row_sync<NT>();
#pragma unroll 1
  for (int i = tid, b = 0; i < l.k; i += NT, b++)
    if (gone >> b & 1) l.link[i].x = -1;
  row_sync<NT>();
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// What a wave knows of a row from its entries alone, in double: what is left of a loss between near distributions are differences of
// logarithms. The student's sum is of e^(s (z - top)), cross = sum q (log q - s (z - top)), mass = sum q.
struct Known {
  double sum, mass, cross, rest;
  float top;
  bool any;  // an entry counts, and the teacher has mass
};
__device__ __forceinline__ Known know(const DistillRows& a, int row, const Listed& l) {
  const int lane = threadIdx.x & 63;
  const double s = a.scale;
  Known n;
  n.top = -INFINITY;
  float t_top = -INFINITY;
  bool any = false;
#pragma unroll 1
  for (int i = lane; i < l.k; i += 64) {
    n.top = fmaxf(n.top, (float)l.share[i]);
    t_top = fmaxf(t_top, (float)l.q[i]);
    any |= l.link[i].x >= 0;
  }
  n.any = __ballot(any) != 0;
  n.top = wave_reduce<true>(n.top);
  t_top = wave_reduce<true>(t_top);
  // (Nothing but -infinity: keep the differences from infinity less infinity.)
  const double z0 = n.top == -INFINITY ? 0.0 : (double)n.top * s, t0 = t_top == -INFINITY ? 0.0 : (double)t_top * s;
  double sum = 0.0, t_sum = 0.0, weighed = 0.0;
#pragma unroll 1
  for (int i = lane; i < l.k; i += 64) {
    const double top = l.q[i], z = l.share[i] * s - z0, t = top * s - (a.lse ? (double)a.lse[row] : t0);
    // (+infinity is no probability: NaN also where the normaliser leaves it infinite.)
    const double e = exp(z), q = l.link[i].x < 0 ? 0.0 : top == INFINITY ? NAN : exp(t);
    sum += e;
    t_sum += q;
    weighed += q == 0.0 ? 0.0 : q * (t - z);
    l.share[i] = e;
    l.q[i] = q;
  }
  n.sum = wave_sum(sum);
  t_sum = wave_sum(t_sum);
  weighed = wave_sum(weighed);
  n.rest = 0.0;
  if (a.lse) {
    n.mass = t_sum;
    n.cross = weighed;
    if (t_sum < 1.0) n.rest = 1.0 - t_sum;
  } else {
    // q is each one's share of their sum (a NaN among them is everyone's).
    const double inverse = 1.0 / t_sum;
    n.any = n.any && !(t_sum == 0.0);
    n.mass = 1.0 + 0.0 * t_sum;
    n.cross = weighed * inverse - log_sum(t_sum);
#pragma unroll 1
    for (int i = lane; i < l.k; i += 64) l.q[i] *= inverse;
  }
  return n;
}

// 1 / x of a normal x, to double's precision but for its last bits; NaN stays.
__device__ __forceinline__ double reciprocal(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
  return __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
}

// What the others' gradient takes: grad_j = each e^((z_j - top) s), and a listed column's: ws (to share - q). part: the row takes part.
struct DistillFactors {
  double ws, to;
  float each;
  int part;
};

// e^(the others' maximum's distance from the listed columns'), below 1 whichever is larger. FAST: to a float's ulp, by the hardware's
// exponential, for gradients: few registers beside a row's.
template <bool FAST>
__device__ __forceinline__ double lead_of(const DistillRows& a, const Known& n, float top) {
  const double x = -fabs(((double)top - (double)n.top) * a.scale);
  if (!FAST) return exp(x);
  const double y = x * 1.44269504088896340736;
  const float high = (float)y;
  // (Infinitely far: no rest.)
  const float rest = high > -1000.f ? (float)(y - (double)high) * 0.693147181f : 0.f;
  return (double)__builtin_fmaf(__builtin_amdgcn_exp2f(high), rest, __builtin_amdgcn_exp2f(high));
}
// The factors from the others' maximum and their sum of e^((z - top) s), 0 where there are none.
__device__ __forceinline__ DistillFactors distill_row(const DistillRows& a, int row, const Known& n, float top, double lead, double total,
                                                      double& all) {
  // (A sum that is NaN takes part, and makes everything NaN.)
  const bool others = !(total == 0.0), listed = n.top != -INFINITY, ahead = others && (!listed || top >= n.top);
  const double mine = !ahead ? 1.0 : listed ? lead : 0.0, theirs = !others ? 0.0 : ahead ? 1.0 : lead;  // of the larger maximum
  all = n.sum * mine + (others ? total * theirs : 0.0);
  DistillFactors f = {0.0, 0.0, 0.f, n.any && !(all == 0.0)};
  if (f.part) {
    f.ws = (a.weight ? (double)a.weight[row] : 1.0) * a.scale;
    const double inverse = reciprocal(all), rest = others ? n.rest : 0.0, mass = n.mass + rest;
    if (others) f.each = (float)(f.ws * (mass * (theirs * inverse) - (rest > 0.0 ? rest * reciprocal(total) : 0.0)));
    f.to = mass * (mine * inverse);
  }
  return f;
}
__device__ __forceinline__ float hot_of(DistillFactors f, double share, double q) { return (float)(f.ws * (f.to * share - q)); }
// The row's loss.
__device__ __forceinline__ float loss_of(const DistillRows& a, int row, const Known& n, float top, double total, double all, bool part) {
  double loss = 0.0;
  if (part) {
    const bool others = !(total == 0.0), listed = n.top != -INFINITY;
    const double s = a.scale, above = others && (!listed || top >= n.top) ? (double)top * s : (double)n.top * s;
    const double lse = above + log_sum(all);
    loss = n.cross + n.mass * (lse - (listed ? (double)n.top * s : 0.0));
    if (others && n.rest > 0.0) loss += n.rest * (log_sum(n.rest) - ((double)top * s + log_sum(total) - lse));
    loss *= a.weight ? (double)a.weight[row] : 1.0;
  }
  return (float)loss;
}

// Rows shorter than 16 bytes: a wave a row, a lane a column.
template <typename T>
__global__ __launch_bounds__(64) void distill_short_kernel(DistillRows a) {
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x;
  const Listed l(lds, a.k);
  const Base2 c2(a.scale);
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const unsigned char* legal = a.legal ? a.legal + (size_t)row * a.ld_legal : nullptr;
    row_sync<64>();  // (the last row's lists have been read)
    l.heads[lane] = 0;
    row_sync<64>();
    list_row<T, 64>(a, row, z, legal, l, Entry(a, row, lane), [](int c) { return c; });
    int mine = -1;  // the entry that lists this lane's column
    for (int h = l.heads[lane]; h; h = l.link[h - 1].y)
      if (l.link[h - 1].x >= 0) mine = h - 1;
    const Known known = know(a, row, l);
    const bool in = lane < a.columns && (!legal || legal[lane]) && mine < 0;
    const float v = in ? (float)z[lane] : -INFINITY, top = wave_reduce<true>(v);
    const float e = exp_of(v - (top == -INFINITY ? 0.f : top), c2);
    const double total = (double)wave_reduce<false>(e);
    double all;
    const DistillFactors f = distill_row(a, row, known, top, lead_of<false>(a, known, top), total, all);
    const float loss = loss_of(a, row, known, top, total, all, f.part);
    if (lane == 0) a.loss[row] = loss;
    if (a.grad && lane < a.columns)
      ((T*)a.grad)[(size_t)row * a.ld_grad + lane] = to_t<T>(!f.part ? 0.f : mine >= 0 ? hot_of(f, l.share[mine], l.q[mine]) : e == 0.f ? 0.f : e * f.each);
  }
}

// w with element j (known at run time) replaced: the element's bits are in each place of `bits` that it can have in a word.
template <typename T>
__device__ __forceinline__ u32x4 replaced(const u32x4& w, int j, unsigned bits) {
  const int k = sizeof(T) == 4 ? j : j >> 1;
  const unsigned mask = sizeof(T) == 4 ? ~0u : j & 1 ? 0xffff0000u : 0xffffu, put = bits & mask;
  return u32x4{k == 0 ? (w[0] & ~mask) | put : w[0], k == 1 ? (w[1] & ~mask) | put : w[1], k == 2 ? (w[2] & ~mask) | put : w[2],
               k == 3 ? (w[3] & ~mask) | put : w[3]};
}
template <typename T>
__device__ __forceinline__ unsigned bits_of(float v) {
  if constexpr (sizeof(T) == 4) return __float_as_uint(v);
  else return __builtin_bit_cast(unsigned short, to_t<T>(v)) * 0x10001u;
}

// An entry's link once its row's chunks are laid: its chunk (-1 where it does not count), and 1 + the next entry with its element of the
// chunk above. A chunk's walk then asks for nothing else.
template <typename T>
__device__ __forceinline__ int2 placed(const Chunks<T>& at, int column, int next) {
  if (column < 0) return int2{-1, next};
  const int c = at.of(column);
  return int2{c, next | (column - at.start(c)) << 16};
}
template <typename T>
__device__ __forceinline__ void place_row(const Lists& l, const Chunks<T>& at) {
#pragma unroll 1
  for (int i = threadIdx.x & 63; i < l.k; i += 64) l.link[i] = placed<T>(at, l.link[i].x, l.link[i].y);
  row_sync<64>();
}

// -infinity in the place of listed columns, of the E chunks of a thread from chunk c0 on.
template <typename T, int NT, int E, int SLOTS = NT * E>
__device__ __forceinline__ void remove_listed(const Lists& l, int tid, const Chunks<T>& at, u32x4 (&raw)[E], int c0) {
  int head[E];
  tid = fresh(tid);
#pragma unroll
  for (int e = 0; e < E; e++) head[e] = l.heads[tid + e * NT % SLOTS];
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (at.none(c0 + e * NT)) break;
    const int c = tid + c0 + e * NT;
    for (int h = head[e]; h; ) {
      const int2 entry = l.link[h - 1];
      if (entry.x == c) raw[e] = replaced<T>(raw[e], entry.y >> 16, bits_of<T>(-INFINITY));
      h = entry.y & 0xffff;
    }
  }
}

// Stores the gradients f of chunk c, of head `slot`, with those of its listed columns.
template <typename T>
__device__ __forceinline__ void store_listed(T* row, const Lists& l, int slot, int c, bool whole, int past, const Chunks<T>& at,
                                             const float (&f)[kVec<T>]) {
  typedef typename AnyWords<T>::type words_t;
  u32x4 w = words_of<T>(f);
  for (int h = l.heads[slot]; h; ) {
    const int2 entry = l.link[h - 1];
    if (entry.x == c) w = replaced<T>(w, entry.y >> 16, bits_of<T>(l.hot[h - 1]));
    h = entry.y & 0xffff;
  }
  const int first = whole ? 0 : at.first(c), limit = whole ? kVec<T> : at.limit(c);
  T* p = row + at.start(c);
  if (whole || (first == 0 && limit == kVec<T>)) {
    if (past) {
      asm volatile("");  // (or the two stores become one, a plain one)
      __builtin_nontemporal_store((words_t)w, (words_t*)p);
      asm volatile("");
    } else {
      *(words_t*)p = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kVec<T>; j++)
      if (j >= first && j < limit) {
        if constexpr (sizeof(T) == 4) ((unsigned*)p)[j] = w[j];
        else ((unsigned short*)p)[j] = (unsigned short)(w[j >> 1] >> (j & 1 ? 16 : 0));
      }
  }
}

// The gradients of a chunk's columns, listed ones aside: each e^((z - base) s).
struct OtherGradients {
  float base, shift, each, factor;
  bool plain;
  Base2 c2;
  // Mostly (z - base) log2 e as one multiply-add: what base log2 e's rounding makes of every term goes into the factor. Not where base is
  // so large that this is a factor of its own, and not where the factor is no number, which columns without mass do not take.
  __device__ __forceinline__ OtherGradients(float base_, float each_, Base2 c) : base(base_), shift(base_ * c.hi), each(each_), c2(c) {
    factor = each * __builtin_amdgcn_exp2f(__builtin_fmaf(-base, c.hi, shift));
    plain = __builtin_amdgcn_readfirstlane(fabsf(shift) < 0x1p20f && fabsf(each) < INFINITY);
  }
  template <typename T>
  __device__ __forceinline__ void of(const u32x4& raw, float (&f)[kVec<T>]) const {
    if (plain) {
#pragma unroll
      for (int j = 0; j < kVec<T>; j++) f[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(element<T>(raw, j), c2.hi, -shift)) * factor;
    } else {
#pragma unroll
      for (int j = 0; j < kVec<T>; j++) {
        const float ex = __builtin_amdgcn_exp2f((element<T>(raw, j) - base) * c2.hi);
        f[j] = ex == 0.f ? 0.f : ex * each;
      }
    }
  }
};

// The maximum of a thread's chunks, their sum of e^((z - top) s) and their gradients, of rows that stay in registers.
template <typename T, int NT, int E>
__device__ __forceinline__ float own_top(const Chunks<T>& at, const u32x4 (&raw)[E]) {
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (at.none(e * NT)) break;
#pragma unroll
    for (int j = 0; j < kVec<T>; j++) top = fmaxf(top, element<T>(raw[e], j));
    __builtin_amdgcn_sched_barrier(0);
  }
  return top;
}
template <typename T, int NT, int E>
__device__ __forceinline__ float own_sum(const Chunks<T>& at, u32x4 (&raw)[E], float base, Base2 c2) {
  forget<E>(raw);
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (at.none(e * NT)) break;
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < kVec<T>; j++) t += exp_of(element<T>(raw[e], j) - base, c2);
    sum += t;
    asm volatile("" : "+v"(sum));  // (here, and not behind the sum's reduction)
    __builtin_amdgcn_sched_barrier(0);
  }
  return sum;
}
template <typename T, int NT, int E, int SLOTS = NT * E>
__device__ __forceinline__ void own_gradient(T* g, int tid, const Chunks<T>& at, u32x4 (&raw)[E], const Lists& l, float base, Base2 c2,
                                             float each, int takes, int past) {
  forget<E>(raw);
  const bool part = __builtin_amdgcn_readfirstlane(takes);
  const OtherGradients others(base, each, c2);
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (at.none(e * NT)) break;
    const int c = fresh(tid) + e * NT;
    float gf[kVec<T>];
    if (part) {
      others.of<T>(raw[e], gf);  // (a listed column's place is filled below)
      store_listed<T>(g, l, tid + e * NT % SLOTS, c, at.whole(e * NT, NT), past, at, gf);
    } else {
      const float zero = __int_as_float(fresh(0));  // (four registers of zeros over the loop of rows are spilled)
#pragma unroll
      for (int j = 0; j < kVec<T>; j++) gf[j] = zero;
      store_gradient<T>(g, c, at.whole(e * NT, NT), past, at, gf);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Rows of up to 64 E chunks: a wave a row, one read.
template <typename T, int E>
__global__ __launch_bounds__(256) void distill_wave_kernel(DistillRows a) {
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x & 63;
  const Listed l(lds + wave_row<64>() * a.list_bytes, a.k);
  const Base2 c2(a.scale);
  for (int row = blockIdx.x * 4 + wave_row<64>(); row < a.rows; row += gridDim.x * 4) {
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const unsigned char* legal = a.legal ? a.legal + (size_t)row * a.ld_legal : nullptr;
    T* g = a.grad ? (T*)a.grad + (size_t)row * a.ld_grad : nullptr;
    const Chunks<T> at(a.columns, g ? g : z);
    u32x4 raw[E], unused[1];
    const Entry mine(a, row, tid);
    load_row<T, 64, E>(z, tid, at, raw);
    row_sync<64>();  // (the last row's lists have been read)
#pragma unroll
    for (int e = 0; e < E; e++) l.heads[tid + e * 64] = 0;
    row_sync<64>();
    list_row<T, 64>(a, row, z, legal, l, mine, [&](int c) { return at.of(c); });
    const Known known = know(a, row, l);
    place_row<T>(l, at);
    if (legal) remove_illegal<T, 64, E, false>(legal, tid, at, raw, unused);
    remove_past<T, 64, E>(tid, at, raw);
    remove_listed<T, 64, E>(l, tid, at, raw, 0);
    const float top = wave_reduce<true>(own_top<T, 64, E>(at, raw)), base = top == -INFINITY ? 0.f : top;
    const double total = (double)wave_reduce<false>(own_sum<T, 64, E>(at, raw, base, c2));
    double all;
    const DistillFactors f = distill_row(a, row, known, top, lead_of<false>(a, known, top), total, all);
#pragma unroll 1
    for (int i = tid; i < l.k; i += 64) l.hot[i] = hot_of(f, l.share[i], l.q[i]);
    row_sync<64>();
    if (g) own_gradient<T, 64, E>(g, tid, at, raw, l, base, c2, f.each, f.part, a.past);
    const float loss = loss_of(a, row, known, top, total, all, f.part);
    if (tid == 0) a.loss[row] = loss;
  }
}

// What the workgroups of longer rows need of the entries, by a wave a row. (Its double arithmetic and its dependent loads in the row's own
// launch, at 4093 x 32768 bf16: 240 us, and 175 by a wave of its own beside the row's; apart 112, 10 of them here.)
constexpr int kSlots = 256;
template <typename T>
__device__ __forceinline__ void know_row(const DistillRows& a, int row, const Listed& l) {
  const int lane = threadIdx.x & 63;
  const Entry mine(a, row, lane);
  row_sync<64>();  // (the last row's lists have been read)
#pragma unroll
  for (int i = 0; i < kSlots / 64; i++) l.heads[lane + i * 64] = 0;
  row_sync<64>();
  list_row<T, 64>(a, row, (const T*)a.logits + (size_t)row * a.ld, a.legal ? a.legal + (size_t)row * a.ld_legal : nullptr, l, mine,
                  [](int c) { return c % kSlots; });
  const Known known = know(a, row, l);
  if (lane == 0) a.known[row] = known;
  for (int i = lane; i < a.k; i += 64) {
    const size_t at = (size_t)row * a.k + i;
    a.column[at] = l.link[i].x;
    a.share[at] = l.share[i];
    a.q[at] = l.q[i];
  }
}
template <typename T>
__global__ __launch_bounds__(64) void distill_known_kernel(DistillRows a) {
  extern __shared__ __align__(16) char lds[];
  const Listed l(lds, a.k);
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) know_row<T>(a, row, l);
}

// What a row's workgroup has of its entries in LDS, copied there by NT threads that ask for theirs before they ask for the row, as what is
// asked for first arrives first. Two barriers around begin(): the last row's are read, and these are there.
struct Copied : Listed {
  Known* known;
  __device__ __forceinline__ Copied(char* lds, int k_) : Listed(lds + sizeof(Known), k_) { known = (Known*)lds; }
  static size_t bytes(int slots, int k) { return (sizeof(Known) + Listed::bytes(slots, k) + 15) / 16 * 16; }
};
template <int NT>
__device__ __forceinline__ int row_thread() { return NT == 64 ? threadIdx.x & 63 : threadIdx.x; }
template <int NT>
struct Asked {
  int c;
  double share, q;
  unsigned known;
  __device__ __forceinline__ Asked(const DistillRows& a, int row) {
    const int i = row_thread<NT>();
    const size_t at = (size_t)row * a.k + min(i, a.k - 1);
    c = a.column[at];
    share = a.share[at];
    q = a.q[at];
    __builtin_memcpy(&known, (const char*)(a.known + row) + min(i, (int)(sizeof(Known) / 4) - 1) * 4, 4);
  }
  __device__ __forceinline__ void begin(const DistillRows& a, int row, const Copied& l) const {
    const int tid = row_thread<NT>();
    if (tid < (int)(sizeof(Known) / 4)) __builtin_memcpy((char*)l.known + tid * 4, &known, 4);
#pragma unroll 1
    for (int i = tid; i < l.k; i += NT) {
      const size_t at = (size_t)row * a.k + i;
      l.share[i] = i == tid ? share : a.share[at];
      l.q[i] = i == tid ? q : a.q[at];
      l.link[i].x = i == tid ? c : a.column[at];
    }
  }
};
// The row's lists, whose heads are 0, from the columns that count: there behind a barrier.
template <typename T, int NT, int SLOTS>
__device__ __forceinline__ void link_row(const Copied& l, const Chunks<T>& at) {
#pragma unroll 1
  for (int i = row_thread<NT>(); i < l.k; i += NT) {
    const int c = l.link[i].x;
    l.link[i] = placed<T>(at, c, c >= 0 ? atomicExch(&l.heads[at.of(c) % SLOTS], i + 1) : 0);
  }
}
template <int NT>
__device__ __forceinline__ void hot_row(const Copied& l, const DistillFactors& f) {
#pragma unroll 1
  for (int i = row_thread<NT>(); i < l.k; i += NT) l.hot[i] = hot_of(f, l.share[i], l.q[i]);
}

// Longer rows that fit the registers of NT threads: a wave a row without a barrier, or a workgroup; one read. (Chunks that are 8 NT apart
// share a list where there are more.)
template <typename T, int NT, int E>
__global__ __launch_bounds__(NT == 64 ? 256 : NT, E > 8 ? 4 : 6) void distill_row_kernel(DistillRows a) {
  constexpr int WAVES = NT / 64, PER = NT == 64 ? 4 : 1, SLOTS = NT * (E < 8 ? E : 8);
  extern __shared__ __align__(16) char lds[];
  __shared__ float tops[WAVES], sums[WAVES];
  __shared__ DistillFactors box;
  const int tid = row_thread<NT>(), wave = NT == 64 ? wave_row<64>() : 0;
  const Copied l(lds + wave * a.list_bytes, a.k);
  const Base2 c2(a.scale);
  for (int row = blockIdx.x * PER + wave; row < a.rows; row += gridDim.x * PER) {
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const unsigned char* legal = a.legal ? a.legal + (size_t)row * a.ld_legal : nullptr;
    T* g = a.grad ? (T*)a.grad + (size_t)row * a.ld_grad : nullptr;
    const Chunks<T> at(a.columns, g ? g : z);
    u32x4 raw[E], unused[1];
    const Asked<NT> asked(a, row);
    load_row<T, NT, E>(z, tid, at, raw);
    row_sync<NT>();
    asked.begin(a, row, l);
#pragma unroll
    for (int e = 0; e < SLOTS / NT; e++) l.heads[tid + e * NT] = 0;
    row_sync<NT>();
    link_row<T, NT, SLOTS>(l, at);
    if (legal) remove_illegal<T, NT, E, false>(legal, tid, at, raw, unused);
    remove_past<T, NT, E>(tid, at, raw);
    row_sync<NT>();
    remove_listed<T, NT, E, SLOTS>(l, tid, at, raw, 0);
    float top = wave_reduce<true>(own_top<T, NT, E>(at, raw));
    if constexpr (NT > 64) {
      if ((tid & 63) == 0) tops[tid >> 6] = top;
      lds_barrier();
#pragma unroll
      for (int k = 0; k < WAVES; k++) top = fmaxf(top, tops[k]);
    }
    const float base = top == -INFINITY ? 0.f : top, sum = wave_reduce<false>(own_sum<T, NT, E>(at, raw, base, c2));
    double total = (double)sum;
    if constexpr (NT > 64) {
      if ((tid & 63) == 0) sums[tid >> 6] = sum;
      lds_barrier();
    }
    DistillFactors f = {};
    if (NT == 64 || tid < 64) {
      const Known known = *l.known;
      if constexpr (NT > 64) {
        total = 0.0;
#pragma unroll
        for (int k = 0; k < WAVES; k++) total += (double)sums[k];
      }
      double all;
      f = distill_row(a, row, known, top, lead_of<true>(a, known, top), total, all);
      if (tid == 0) {
        if (NT > 64) box = f;
        a.others[row] = Others{total, top};
      }
    }
    if constexpr (NT > 64) lds_barrier();
    const DistillFactors& shared = NT > 64 ? box : f;
    hot_row<NT>(l, shared);
    row_sync<NT>();
    if (g) own_gradient<T, NT, E, SLOTS>(g, tid, at, raw, l, base, c2, shared.each, shared.part, a.past);
  }
}

// A row's loss from what the launches before found, by one thread. (At the end of a row's own launch its constants alone, which the
// compiler keeps over the loop of rows, cost 50 registers a thread.)
__device__ __forceinline__ void loss_row(const DistillRows& a, int row, const Others& others) {
  const Known known = a.known[row];
  double all;
  const DistillFactors f = distill_row(a, row, known, others.top, lead_of<false>(a, known, others.top), others.total, all);
  a.loss[row] = loss_of(a, row, known, others.top, others.total, all, f.part);
}
__global__ __launch_bounds__(64) void distill_loss_kernel(DistillRows a) {
  for (int row = blockIdx.x * 64 + threadIdx.x; row < a.rows; row += gridDim.x * 64) loss_row(a, row, a.others[row]);
}
// The same from the rows' parts.
__device__ __forceinline__ void losses_of_parts(const DistillRows& a, int first, int step, Base2 c2) {
  for (int row = first; row < a.rows; row += step) {
    const Others* parts = a.parts + (size_t)row * a.split;
    Others others = {0.0, -INFINITY};
    for (int k = 0; k < a.split; k++) others.top = fmaxf(others.top, parts[k].top);
    for (int k = 0; k < a.split; k++)
      others.total += parts[k].top == -INFINITY ? parts[k].total : parts[k].total * (double)exp_of(parts[k].top - others.top, c2);
    loss_row(a, row, others);
  }
}

// Longer rows: E chunks of each thread at a time relative to the running maximum, and again for the gradient, whose second reading comes
// from the caches. Few such rows are cut into parts for as many workgroups: a launch for the parts' sums (PARTS), and one that joins
// them and writes the gradient (JOIN): 301 rows of 100003 f16 62 us whole, 44 in parts (a call 49 with the entries in a launch
// before, 45 with workgroups for them ahead of the parts').
enum { WHOLE, PARTS, JOIN };
constexpr int kKnowing = 4;
template <typename T, int NT, int E, int STAGE>
__global__ __launch_bounds__(NT) void distill_long_kernel(DistillRows a) {
  constexpr int V = kVec<T>, SLOTS = NT * E;
  extern __shared__ __align__(16) char lds[];
  __shared__ float red[16];
  __shared__ DistillFactors box;
  __shared__ float base;
  const int tid = threadIdx.x;
  const Copied l(lds, a.k);
  const Base2 c2(a.scale);
  // (The launch that joins has a workgroup more, for the losses.)
  if (STAGE == JOIN && blockIdx.x + 1 == gridDim.x) {
    losses_of_parts(a, tid, NT, c2);
    return;
  }
  if (STAGE == PARTS && (int)blockIdx.x < a.knowing) {
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (wave < kKnowing)
      for (int row = blockIdx.x * kKnowing + wave; row < a.rows; row += a.knowing * kKnowing) know_row<T>(a, row, Listed(lds + wave * a.list_bytes, a.k));
    return;
  }
  for (int id = blockIdx.x - (STAGE == PARTS ? a.knowing : 0); id < a.rows * (STAGE == WHOLE ? 1 : a.split); id += gridDim.x - (STAGE == JOIN)) {
    const int row = STAGE == WHOLE ? id : id / a.split, part = STAGE == WHOLE ? 0 : id - row * a.split;
    const int begin = part * a.span, end = STAGE == WHOLE ? INT_MAX : begin + a.span;  // its chunks, whole pieces of SLOTS
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const unsigned char* legal = a.legal ? a.legal + (size_t)row * a.ld_legal : nullptr;
    T* g = a.grad ? (T*)a.grad + (size_t)row * a.ld_grad : nullptr;
    const Chunks<T> at(a.columns, g ? g : z);
    if (STAGE == PARTS) {  // (whether an entry counts is not asked: an illegal column is not among the others either)
      lds_barrier();
      for (int i = tid; i < l.k; i += NT) {
        const int c = a.index[(size_t)row * a.ld_index + i];
        l.link[i].x = (unsigned)c < (unsigned)a.columns ? c : -1;
      }
    } else {
      const Asked<NT> asked(a, row);
      lds_barrier();
      asked.begin(a, row, l);
    }
#pragma unroll
    for (int e = 0; e < E; e++) l.heads[tid + e * NT] = 0;
    lds_barrier();
    link_row<T, NT, SLOTS>(l, at);
    lds_barrier();
    auto piece = [&](int c0, u32x4(&raw)[E]) {
      u32x4 unused[1];
      load_row<T, NT, E>(z, tid, at, raw, c0);
      if (legal) remove_illegal<T, NT, E, false>(legal, tid, at, raw, unused, c0);
      remove_past<T, NT, E>(tid, at, raw, c0);
    };
    Running run;
    if (STAGE != JOIN) {
      for (int c0 = begin; c0 < end && !at.none(c0); c0 += SLOTS) {
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
    }
    if (STAGE == PARTS) {
      if (tid == 0) a.parts[id] = Others{run.total, run.top};
      continue;
    }
    if (tid < 64) {
      if (STAGE == JOIN) {
        Others q = {0.0, -INFINITY};
        if (tid < a.split) q = a.parts[row * a.split + tid];
        run.top = wave_reduce<true>(q.top);
        run.total = wave_sum(q.top == -INFINITY ? q.total : q.total * (double)exp_of(q.top - run.top, c2));
      }
      const Known known = *l.known;
      double all;
      const DistillFactors f = distill_row(a, row, known, run.top, lead_of<true>(a, known, run.top), run.total, all);
      if (tid == 0) {
        box = f;
        base = run.top == -INFINITY ? 0.f : run.top;
        if (STAGE == WHOLE) a.others[row] = Others{run.total, run.top};
      }
    }
    lds_barrier();
    if (!g) continue;
    hot_row<NT>(l, box);
    lds_barrier();
    const bool takes = __builtin_amdgcn_readfirstlane(box.part);
    const OtherGradients others(base, box.each, c2);
    for (int c0 = begin; c0 < end && !at.none(c0); c0 += SLOTS) {
      u32x4 raw[E];
      if (takes) piece(c0, raw);
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (at.none(c0 + e * NT)) break;
        const int c = fresh(tid) + c0 + e * NT;
        float gf[V] = {};
        if (takes) {
          others.of<T>(raw[e], gf);  // (a listed column's place is filled below)
          store_listed<T>(g, l, tid + e * NT, c, at.whole(c0 + e * NT, NT), a.past, at, gf);
        } else {
          store_gradient<T>(g, c, at.whole(c0 + e * NT, NT), a.past, at, gf);
        }
      }
    }
  }
}

// Rows that a wave takes alone, whatever their type: they need no workspace, as the header promises.
constexpr int kWaveColumns = 448, kWaveEntries = 256;

template <typename T>
void distill_typed(DistillRows p, hipStream_t s) {
  const dim3 groups(row_grid(p.rows, 1));
  if (p.columns < kVec<T>) return launch_k(distill_short_kernel<T>, groups, 64, Listed::bytes(64, p.k), s, p);
  const RowShape r = p.grad ? row_shape<T>(p.columns, p.grad, p.ld_grad, p.rows) : row_shape<T>(p.columns, p.logits, p.ld, p.rows);
  if (r.threads == 64 && r.each == 2 && p.k <= kWaveEntries) {
    p.list_bytes = (int)Listed::bytes(64 * 2, p.k);
    return launch_k(distill_wave_kernel<T, 2>, dim3(row_grid(p.rows, 4)), 256, p.list_bytes * 4, s, p);
  }
  const RowParts cut = r.threads == 0 ? row_parts<T>(p.rows, p.columns, 512 * 4) : RowParts{1, 0};
  if (cut.split > 1) {
    const size_t lds = Copied::bytes(512 * 4, p.k);
    p.split = cut.split;
    p.span = cut.span;
    p.list_bytes = (int)Listed::bytes(kSlots, p.k);
    // (With few entries each row's are known beside the parts, which take the listed columns as they stand.)
    if (p.k <= kWaveEntries) p.knowing = (p.rows + kKnowing - 1) / kKnowing;
    else launch_k(distill_known_kernel<T>, groups, 64, p.list_bytes, s, p);
    launch_k(distill_long_kernel<T, 512, 4, PARTS>, dim3(p.rows * p.split + p.knowing), 512, std::max(lds, (size_t)p.list_bytes * (p.knowing ? kKnowing : 0)), s, p);
    return launch_k(distill_long_kernel<T, 512, 4, JOIN>, dim3(p.grad ? p.rows * p.split + 1 : 1), 512, lds, s, p);
  }
  launch_k(distill_known_kernel<T>, groups, 64, Listed::bytes(kSlots, p.k), s, p);
  if (r.threads == 64 && p.k <= kWaveEntries) {
    p.list_bytes = (int)Copied::bytes(64 * 8, p.k);
    launch_k(distill_row_kernel<T, 64, 8>, dim3(row_grid(p.rows, 4)), 256, p.list_bytes * 4, s, p);
  } else if (r.threads == 64) launch_k(distill_row_kernel<T, 256, 2>, groups, 256, Copied::bytes(256 * 2, p.k), s, p);
  else if (r.threads == 256) launch_k(distill_row_kernel<T, 256, 8>, groups, 256, Copied::bytes(256 * 8, p.k), s, p);
  else if (r.threads == 512) launch_k(distill_row_kernel<T, 512, 8>, groups, 512, Copied::bytes(512 * 8, p.k), s, p);
  else {
    // (As many chunks a thread again where rows are not cut: 4093 x 33000 bf16 204 us by pieces, 167 held, 2048 x 50257 bf16 151 and 136; but
    // 300 x 50257 floats 58 in parts, 61 held, and rows twice as long by 1024 threads 325 where pieces take 313.)
    const long long chunks = ((long long)p.columns + kVec<T> - 1) / kVec<T> + Chunks<T>::line(p.columns) / 16;
    if (chunks <= 512 * 16) launch_k(distill_row_kernel<T, 512, 16>, groups, 512, Copied::bytes(512 * 8, p.k), s, p);
    else launch_k(distill_long_kernel<T, 512, 4, WHOLE>, groups, 512, Copied::bytes(512 * 4, p.k), s, p);
  }
  launch_k(distill_loss_kernel, dim3(row_grid(p.rows, 64)), 64, 0, s, p);
}

// Where what is known of the entries lies in the workspace.
struct Plan {
  size_t known, others, parts, share, q, column, bytes;
};
Plan plan_of(int rows, int columns, int k) {
  Plan p = {};
  const auto room = [&](size_t n) {
    const size_t at = p.bytes;
    p.bytes += (n + 255) / 256 * 256;
    return at;
  };
  p.known = room((size_t)rows * sizeof(Known));
  p.others = room((size_t)rows * sizeof(Others));
  p.parts = room((size_t)rows * most_parts(rows, columns) * sizeof(Others));
  p.share = room((size_t)rows * k * 8);
  p.q = room((size_t)rows * k * 8);
  p.column = room((size_t)rows * k * 4);
  return p;
}

}  // namespace

size_t distill_loss_workspace(int rows, int columns, int k) {
  if (rows < 1 || k < 1 || (columns <= kWaveColumns && k <= kWaveEntries)) return 0;
  return plan_of(rows, columns, k).bytes;
}

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
  const Plan plan = plan_of(a.rows, a.columns, a.k);
  char* w = (char*)a.workspace;
  p.known = (Known*)(w + plan.known);
  p.others = (Others*)(w + plan.others);
  p.parts = (Others*)(w + plan.parts);
  p.split = 1;
  p.span = 0;
  p.knowing = 0;
  p.share = (double*)(w + plan.share);
  p.q = (double*)(w + plan.q);
  p.column = (int*)(w + plan.column);
  switch (a.type) {
    case PREC_F32: distill_typed<float>(p, s); break;
    case PREC_F16: distill_typed<f16>(p, s); break;
    default: distill_typed<bf16>(p, s); break;
  }
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
