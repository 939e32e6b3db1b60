// The policy and preference losses with their gradients (kg_policy_loss, kg_preference_loss).
//
// Both are softmax cross-entropies whose gradient factor depends on the whole row (the clip, the KL term) or on whole
// sequences (the margin): a row's maximum, sum and chosen log-probability come first, then grad = factor (onehot - p), plus
// the KL term's p (log p/r - KL). One pass over a row keeps the running maximum and the sum of exp relative to it; with a
// reference row also the reference's and sum e^(z - max) ((z - max) - (r - max_r)), from which KL = sum p ((z - max) -
// (r - max_r)) - log(sum / sum_r) follows without a second look (both rows relative to their maxima: no cancellation
// between rows far from 0, and none with a mask of the type's lowest value). A second pass writes the gradient.
//
// A row's few scalars are computed in double: logp decides on which side of the clip the row is, and the losses of a
// sequence are differences of sums of thousands. (A comparison of logp - old_logp with log(1 +- clip) needs no exp.)
#include <algorithm>
#include <climits>

#include "kgx_device.h"
#include "kgx_learn.h"
#include "kgx_rows.h"

namespace kgx {

namespace {

// The sums over a part of a row (see PolicyRows), relative to the part's maxima.
struct PolicyPart {
  double sum, ref_sum;
  float top, ref_top, cross, none;
};
struct PolicyRows {
  const void* logits;
  const unsigned char* legal;
  const void* ref;
  void* grad;
  long long ld, ld_legal, ld_ref, ld_grad;
  const int* action;
  const float *old_logp, *advantage, *weight, *ref_logp;
  float *loss, *logp, *kl;
  PolicyPart* parts;  // rows cut into `split` parts of `span` chunks (1: not cut)
  int rows, columns, past, split, span;
  double scale, low, high, log_low, log_high;  // clip_low, clip_high; log(1 - clip_low), log(1 + clip_high)
  float kl_coef;
};

// What a row's gradient takes from its sums: grad_j = e_j (f_p + f_kl (d_j - shift)) with e_j = e^((z_j - top) s) and d_j the
// difference of z - top and the reference's, times s; plus hot at the action. part: the row takes part.
struct PolicyFactors {
  float hot, f_p, f_kl, shift;
  int part;
};

// The row's results and factors from its sums, the action's logit (-infinity where it is illegal) and cross = sum e^(z -
// top) ((z - top) - (r - its top)). Every lane of a wave computes them; `writes`: this one stores the results.
template <bool FULL>
__device__ __forceinline__ PolicyFactors policy_row(const PolicyRows& a, int row, bool padding, float za, float top, double sum,
                                                    double ref_sum, float cross, bool writes) {
  const double log_s = log_sum(sum);
  const double lp = za == -INFINITY ? -(double)INFINITY : ((double)za - (double)top) * a.scale - log_s;
  PolicyFactors f = {0.f, 0.f, 0.f, 0.f, !padding && !(lp == -(double)INFINITY)};
  float loss = 0.f, logp = padding ? 0.f : -INFINITY, kl = 0.f;
  if (f.part) {
    // (1 / sum by the hardware's reciprocal: an ulp of the row's probabilities, whose exponentials are off by more.)
    const float w = a.weight ? a.weight[row] : 1.f, adv = a.advantage[row], inv = __builtin_amdgcn_rcpf((float)sum);
    const double delta = lp - (double)a.old_logp[row];
    const float ratio = exp_of((float)delta, Base2(1.0));
    // (No advantage: 0 on either side, and on the held one whatever the ratio. NaN is on neither.)
    const bool held = adv >= 0.f ? delta > a.log_high : adv < 0.f ? delta < a.log_low : false;
    const float bounded = fminf(fmaxf(ratio, (float)(1.0 - a.low)), (float)(1.0 + a.high));
    float c = held ? 0.f : -ratio * adv;
    if constexpr (FULL) {
      const double gap = log_s - log_sum(ref_sum);
      const double k = (double)cross * a.scale * (double)inv - gap;
      kl = (float)k;
      f.shift = (float)(gap + k);
    } else if (a.ref_logp) {
      const float d = (float)((double)a.ref_logp[row] - lp), em = expm1f(d);
      kl = em - d;
      c -= a.kl_coef * em;
    }
    const float gw = w * (float)a.scale;
    f.hot = gw * c;
    f.f_p = -f.hot * inv;
    f.f_kl = FULL ? a.kl_coef * gw * inv : 0.f;
    loss = w * (a.kl_coef * kl - (held ? bounded : ratio) * adv);
    logp = (float)lp;
  }
  if (writes) {
    a.loss[row] = loss;
    a.logp[row] = logp;
    a.kl[row] = kl;
  }
  return f;
}

// The same for a row of NT threads: one wave computes, the others read its factors.
template <int NT, bool FULL>
__device__ __forceinline__ PolicyFactors policy_row_shared(const PolicyRows& a, int row, float za, float top, double sum,
                                                           double ref_sum, float cross, PolicyFactors* box) {
  if constexpr (NT <= 64) {
    return policy_row<FULL>(a, row, false, za, top, sum, ref_sum, cross, (threadIdx.x & 63) == 0);
  } else {
    if (threadIdx.x < 64) {
      const PolicyFactors f = policy_row<FULL>(a, row, false, za, top, sum, ref_sum, cross, threadIdx.x == 0);
      if (threadIdx.x == 0) *box = f;
    }
    lds_barrier();
    return *box;  // (the next row's reductions lie between this and the next writing)
  }
}

// Rows shorter than 16 bytes: a wave a row, a lane a column.
template <typename T, bool FULL, bool LEGAL>
__global__ __launch_bounds__(256) void policy_short_kernel(PolicyRows a) {
  const int lane = threadIdx.x & 63;
  const Base2 c2(a.scale);
  for (int row = blockIdx.x * 4 + wave_row<64>(); row < a.rows; row += gridDim.x * 4) {
    const int act = a.action[row];
    const bool padding = (unsigned)act >= (unsigned)a.columns;
    const bool in = !padding && lane < a.columns && (!LEGAL || a.legal[(size_t)row * a.ld_legal + lane]);
    const float z = in ? (float)((const T*)a.logits)[(size_t)row * a.ld + lane] : -INFINITY;
    float top = wave_reduce<true>(z), x = 0.f, ref_sum = 0.f, cross = 0.f;
    if (top == -INFINITY) top = 0.f;
    const float e = exp_of(z - top, c2);
    if constexpr (FULL) {
      const float r = in ? (float)((const T*)a.ref)[(size_t)row * a.ld_ref + lane] : -INFINITY;
      float ref_top = wave_reduce<true>(r);
      if (ref_top == -INFINITY) ref_top = 0.f;
      ref_sum = wave_reduce<false>(exp_of(r - ref_top, c2));
      x = (z - top) - (r - ref_top);
      cross = wave_reduce<false>(e == 0.f ? 0.f : e * x);
    }
    const float sum = wave_reduce<false>(e), za = padding ? -INFINITY : lane_of(z, act);
    const PolicyFactors f = policy_row<FULL>(a, row, padding, za, top, sum, ref_sum, cross, lane == 0);
    if (a.grad && lane < a.columns) {
      float g = 0.f;
      if (f.part && !(FULL && e == 0.f)) g = e * (FULL ? f.f_p + f.f_kl * (x * (float)a.scale - f.shift) : f.f_p);
      if (f.part && lane == act) g += f.hot;
      ((T*)a.grad)[(size_t)row * a.ld_grad + lane] = to_t<T>(g);
    }
  }
}

// Illegal columns and chunk elements past the row become -infinity in the words once, and from there on need no test: their
// exponential is 0, and with it their gradient. Bound by memory, one read and one write: 4093 x 32768 bf16 in 89 us (6 TB/s),
// 16384 x 362 float rows of 1094 with legality and a full KL in 22 (3.5 TB/s); 32 such rows 5.4 us, the latency of one.
template <typename T, int NT, int E, bool FULL, bool LEGAL>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void policy_row_kernel(PolicyRows a) {
  constexpr int V = kVec<T>, PER = NT < 256 ? 256 / NT : 1;
  __shared__ float red[16];
  __shared__ PolicyFactors box;
  const int tid = threadIdx.x % NT;
  const float s = (float)a.scale;
  const Base2 c2(a.scale);
  for (int row = blockIdx.x * PER + wave_row<NT>(); row < a.rows; row += gridDim.x * PER) {
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const unsigned char* lg = LEGAL && a.legal ? a.legal + (size_t)row * a.ld_legal : nullptr;
    T* g = a.grad ? (T*)a.grad + (size_t)row * a.ld_grad : nullptr;
    const Chunks<T> at(a.columns, g ? g : z);
    const int act = a.action[row];
    const bool padding = (unsigned)act >= (unsigned)a.columns;
    PolicyFactors f = {0.f, 0.f, 0.f, 0.f, 0};
    float top = 0.f, ref_top = 0.f;
    u32x4 raw[E], ref[FULL ? E : 1];
    if (!padding) {
      load_row<T, NT, E>(z, tid, at, raw);
      if constexpr (FULL) load_row<T, NT, E>((const T*)a.ref + (size_t)row * a.ld_ref, tid, at, ref);
      float za = (float)z[act];
      if (lg) {
        if (!lg[act]) za = -INFINITY;
        remove_illegal<T, NT, E, FULL>(lg, tid, at, raw, ref);
      }
      remove_past<T, NT, E>(tid, at, raw);
      if constexpr (FULL) remove_past<T, NT, E>(tid, at, ref);
      top = max_of<T, NT, E>(raw, at, red);
      if constexpr (FULL) ref_top = max_of<T, NT, E>(ref, at, red);
      if (top == -INFINITY) top = 0.f;
      if (FULL && ref_top == -INFINITY) ref_top = 0.f;
      float sum = 0.f, ref_sum = 0.f, cross = 0.f;
      forget<E>(raw);
      if constexpr (FULL) forget<E>(ref);
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (at.none(e * NT)) break;
        float t = 0.f, tr = 0.f, tx = 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float x = element<T>(raw[e], j) - top, ex = exp_of(x, c2);
          t += ex;
          if constexpr (FULL) {
            const float rx = element<T>(ref[e], j) - ref_top;
            tr += exp_of(rx, c2);
            tx += ex == 0.f ? 0.f : ex * (x - rx);
          }
        }
        sum += t;
        ref_sum += tr;
        cross += tx;
        // (Here, and not behind the first sum's reduction.)
        asm volatile("" : "+v"(sum), "+v"(ref_sum), "+v"(cross));
        __builtin_amdgcn_sched_barrier(0);
      }
      const double total = row_sum<NT>(sum, red);
      double ref_total = 0.0;
      if constexpr (FULL) {
        ref_total = row_sum<NT>(ref_sum, red);
        cross = row_reduce<NT, false>(cross, red);
      }
      f = policy_row_shared<NT, FULL>(a, row, za, top, total, ref_total, cross, &box);
      forget<E>(raw);
      if constexpr (FULL) forget<E>(ref);
    } else if (tid == 0) {
      a.loss[row] = a.logp[row] = a.kl[row] = 0.f;
    }
    if (!g) continue;
    if (!__builtin_amdgcn_readfirstlane(f.part)) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (at.none(e * NT)) break;
        const float none[V] = {};
        store_gradient<T>(g, fresh(tid) + e * NT, at.whole(e * NT, NT), a.past, at, none);
      }
      continue;
    }
    const int hot_chunk = at.of(act);
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (at.none(e * NT)) break;
      const int c = fresh(tid) + e * NT;
      float gf[V];
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float x = element<T>(raw[e], j) - top, ex = __builtin_amdgcn_exp2f(x * c2.hi);
        float k = f.f_p;
        if constexpr (FULL) k += f.f_kl * ((x - (element<T>(ref[e], j) - ref_top)) * s - f.shift);
        gf[j] = FULL && ex == 0.f ? 0.f : ex * k;
      }
      if (c == hot_chunk) {
        const int hot = act - at.start(c);
#pragma unroll
        for (int j = 0; j < V; j++) gf[j] += j == hot ? f.hot : 0.f;
      }
      store_gradient<T>(g, c, at.whole(e * NT, NT), a.past, at, gf);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Longer rows: E chunks of each thread at a time relative to the running maxima, and again for the gradient, whose second
// reading comes from the caches. (Held by 1024 threads in 16 chunks each, a row has a CU to itself, whose loads,
// exponentials and stores wait for each other.)
// Few such rows are cut into parts for as many workgroups: a launch for the parts' sums (PARTS), and one that joins them and writes
// the gradient (JOIN). One row of 125123 f16 with legality and a full KL took 62 us on one CU, now 10.
enum { WHOLE, PARTS, JOIN };
template <typename T, int NT, int E, bool FULL, bool LEGAL, int STAGE>
__global__ __launch_bounds__(NT) void policy_long_kernel(PolicyRows a) {
  constexpr int V = kVec<T>;
  __shared__ float red[16];
  __shared__ PolicyFactors box;
  __shared__ float tops[2];
  const int tid = threadIdx.x;
  const float s = (float)a.scale;
  const Base2 c2(a.scale);
  for (int id = blockIdx.x; id < a.rows * (STAGE == WHOLE ? 1 : a.split); id += gridDim.x) {
    const int row = STAGE == WHOLE ? id : id / a.split, part = STAGE == WHOLE ? 0 : id - row * a.split;
    const int begin = part * a.span, end = STAGE == WHOLE ? INT_MAX : begin + a.span;  // its chunks
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const T* r = FULL ? (const T*)a.ref + (size_t)row * a.ld_ref : nullptr;
    const unsigned char* lg = LEGAL ? a.legal + (size_t)row * a.ld_legal : nullptr;
    T* g = a.grad ? (T*)a.grad + (size_t)row * a.ld_grad : nullptr;
    const Chunks<T> at(a.columns, g ? g : z);
    const int act = a.action[row];
    const bool padding = (unsigned)act >= (unsigned)a.columns;
    Running run, ref;
    PolicyFactors f = {0.f, 0.f, 0.f, 0.f, 0};
    // The words of E chunks of the row (and of the reference's) from chunk c0 on, with -infinity where nothing is.
    auto piece = [&](int c0, u32x4(&raw)[E], u32x4(&raw_r)[FULL ? E : 1]) {
      load_row<T, NT, E>(z, tid, at, raw, c0);
      if constexpr (FULL) load_row<T, NT, E>(r, tid, at, raw_r, c0);
      if constexpr (LEGAL) remove_illegal<T, NT, E, FULL>(lg, tid, at, raw, raw_r, c0);
      remove_past<T, NT, E>(tid, at, raw, c0);
      if constexpr (FULL) remove_past<T, NT, E>(tid, at, raw_r, c0);
    };
    if (!padding && STAGE != JOIN) {
      float cross = 0.f;
      for (int c0 = begin; c0 < end && !at.none(c0); c0 += NT * E) {
        u32x4 raw[E], raw_r[FULL ? E : 1];
        piece(c0, raw, raw_r);
        float fz[E * V], e[E * V], moved;
#pragma unroll
        for (int k = 0; k < E; k++) {
#pragma unroll
          for (int j = 0; j < V; j++) fz[k * V + j] = !at.none(c0 + k * NT) ? element<T>(raw[k], j) : -INFINITY;
        }
        const float before = run.sum;
        const float keep = run.add<E * V>(fz, c2, e, moved);
        if constexpr (FULL) {
          float fr[E * V], er[E * V], r_moved;
#pragma unroll
          for (int k = 0; k < E; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) fr[k * V + j] = !at.none(c0 + k * NT) ? element<T>(raw_r[k], j) : -INFINITY;
          }
          ref.add<E * V>(fr, c2, er, r_moved);
          float x = 0.f;
#pragma unroll
          for (int j = 0; j < E * V; j++) x += e[j] == 0.f ? 0.f : e[j] * (fz[j] - fr[j]);
          cross = keep == 0.f ? x : __builtin_fmaf(__builtin_fmaf(before, moved - r_moved, cross), keep, x);
        }
      }
      const float before = run.sum;
      float moved, r_moved;
      const float keep = run.join<NT>(c2, red, moved);
      if constexpr (FULL) {
        ref.join<NT>(c2, red, r_moved);
        cross = row_reduce<NT, false>(keep == 0.f ? 0.f : __builtin_fmaf(before, moved - r_moved, cross) * keep, red);
      }
      if constexpr (STAGE == PARTS) {
        if (tid == 0) a.parts[id] = PolicyPart{run.total, ref.total, run.top, ref.top, cross, 0.f};
      } else {
        const float za = !LEGAL || lg[act] ? (float)z[act] : -INFINITY;
        f = policy_row_shared<NT, FULL>(a, row, za, run.top, run.total, ref.total, cross, &box);
      }
    } else if (STAGE == JOIN && !padding) {
      lds_barrier();  // (the last part's factors have been read)
      if (tid < 64) {
        PolicyPart q = {0.0, 0.0, -INFINITY, -INFINITY, 0.f, 0.f};
        if (tid < a.split) q = a.parts[row * a.split + tid];
        const float top = wave_reduce<true>(q.top), ref_top = FULL ? wave_reduce<true>(q.ref_top) : 0.f;
        const float moved = q.top - top, keep = q.top == -INFINITY ? 0.f : exp_of(moved, c2);
        double total = q.sum * (double)keep, ref_total = 0.0;
        float cross = 0.f;
        if constexpr (FULL) {
          const float r_moved = q.ref_top - ref_top;
          ref_total = q.ref_sum * (double)(q.ref_top == -INFINITY ? 0.f : exp_of(r_moved, c2));
          cross = wave_reduce<false>(keep == 0.f ? 0.f : __builtin_fmaf((float)q.sum, moved - r_moved, q.cross) * keep);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
          total += __shfl_xor(total, o);
          if constexpr (FULL) ref_total += __shfl_xor(ref_total, o);
        }
        const float za = !LEGAL || lg[act] ? (float)z[act] : -INFINITY;
        const PolicyFactors mine = policy_row<FULL>(a, row, false, za, top, total, ref_total, cross, tid == 0 && part == 0);
        if (tid == 0) {
          box = mine;
          tops[0] = top;
          tops[1] = ref_top;
        }
      }
      lds_barrier();
      f = box;
      run.top = tops[0];
      ref.top = tops[1];
    } else if (tid == 0 && part == 0) {
      a.loss[row] = a.logp[row] = a.kl[row] = 0.f;
    }
    if (STAGE == PARTS || !g) continue;
    const bool takes = __builtin_amdgcn_readfirstlane(f.part);
    const int hot_chunk = takes ? at.of(act) : -1;
    for (int c0 = begin; c0 < end && !at.none(c0); c0 += NT * E) {
      u32x4 raw[E], raw_r[FULL ? E : 1];
      if (takes) piece(c0, raw, raw_r);
#pragma unroll
      for (int k = 0; k < E; k++) {
        if (at.none(c0 + k * NT)) break;
        const int c = fresh(tid) + c0 + k * NT;
        float gf[V] = {};
        if (takes) {
#pragma unroll
          for (int j = 0; j < V; j++) {
            const float x = element<T>(raw[k], j) - run.top, ex = __builtin_amdgcn_exp2f(x * c2.hi);
            float m = f.f_p;
            if constexpr (FULL) m += f.f_kl * ((x - (element<T>(raw_r[k], j) - ref.top)) * s - f.shift);
            gf[j] = FULL && ex == 0.f ? 0.f : ex * m;
          }
          if (c == hot_chunk) {
            const int hot = act - at.start(c);
#pragma unroll
            for (int j = 0; j < V; j++) gf[j] += j == hot ? f.hot : 0.f;
          }
        }
        store_gradient<T>(g, c, at.whole(c0 + k * NT, NT), a.past, at, gf);
      }
    }
  }
}

template <typename T, bool FULL, bool LEGAL>
void policy_rows(const PolicyRows& p, hipStream_t s) {
  PolicyRows cut = p;
  const RowParts parts = row_parts<T>(p.rows, p.columns, 512 * (FULL ? 2 : 4));
  cut.split = parts.split;
  cut.span = parts.span;
  const RowShape r = p.grad ? row_shape<T>(p.columns, p.grad, p.ld_grad, p.rows) : row_shape<T>(p.columns, p.logits, p.ld, p.rows);
  const dim3 waves(row_grid(p.rows, 4)), groups(row_grid(p.rows, 1));
  if (r.threads == 64 && r.each == 2) launch_k(policy_row_kernel<T, 64, 2, FULL, LEGAL>, waves, 256, 0, s, p);
  else if (r.threads == 64) launch_k(policy_row_kernel<T, 64, 8, FULL, LEGAL>, waves, 256, 0, s, p);
  else if (r.threads == 256) launch_k(policy_row_kernel<T, 256, 8, FULL, LEGAL>, groups, 256, 0, s, p);
  else if (r.threads == 512) launch_k(policy_row_kernel<T, 512, 8, FULL, LEGAL>, groups, 512, 0, s, p);
  else if (p.columns < kVec<T>) launch_k(policy_short_kernel<T, FULL, LEGAL>, waves, 256, 0, s, p);
  // (Float rows over 160 KB on 1024 threads: with four workgroups of 512 a CU, more rows are under way than the caches hold
  // for the second reading: 614 against 477 us with gradient at 2700 x 100000, 431 against 442 at 8192 x 32768. 16-bit rows, half
  // as long, stay on 512: 274 against 292 us.)
  else if (cut.split > 1) {
    const dim3 grid(p.rows * cut.split);
    launch_k(policy_long_kernel<T, 512, FULL ? 2 : 4, FULL, LEGAL, PARTS>, grid, 512, 0, s, cut);
    launch_k(policy_long_kernel<T, 512, FULL ? 2 : 4, FULL, LEGAL, JOIN>, grid, 512, 0, s, cut);
  } else if (sizeof(T) == 4 && p.columns > 40960) launch_k(policy_long_kernel<T, 1024, 2, FULL, LEGAL, WHOLE>, groups, 1024, 0, s, p);
  else launch_k(policy_long_kernel<T, 512, FULL ? 2 : 4, FULL, LEGAL, WHOLE>, groups, 512, 0, s, p);
}

template <typename T>
void policy_typed(const PolicyRows& p, hipStream_t s) {
  if (p.ref) {
    if (p.legal) policy_rows<T, true, true>(p, s);
    else policy_rows<T, true, false>(p, s);
  } else {
    if (p.legal) policy_rows<T, false, true>(p, s);
    else policy_rows<T, false, false>(p, s);
  }
}

// The sum over a part of a row, relative to the part's maximum.
struct PrefPart {
  double sum;
  float top, none;
};
struct PrefRows {
  const void* logits;
  void* grad;
  long long ld, ld_grad;
  const int *label, *offsets;
  const float *ref_logp, *weight;
  PrefRow* row;
  float* coef;
  PrefPart* parts;  // rows cut into `split` parts of `span` chunks (1: not cut)
  int split, span;
  float *loss, *margin, *seq_logp;
  int rows, columns, past, pairs, average;
  double beta, smooth;
};

// Row t's softmax maximum, reciprocal sum and log-probability of its label, where it counts; its gradient's factor starts
// at 0. Here for rows shorter than 16 bytes: a wave a row, a lane a column.
template <typename T>
__global__ __launch_bounds__(256) void pref_rows_short_kernel(PrefRows a) {
  const int lane = threadIdx.x & 63, first = a.offsets[0], last = a.offsets[2 * a.pairs];
  const Base2 c2(1.0);
  for (int row = blockIdx.x * 4 + wave_row<64>(); row < a.rows; row += gridDim.x * 4) {
    const int label = a.label[row];
    if (lane == 0) a.coef[row] = 0.f;
    if (row < first || row >= last || (unsigned)label >= (unsigned)a.columns) continue;
    const float z = lane < a.columns ? (float)((const T*)a.logits)[(size_t)row * a.ld + lane] : -INFINITY;
    float top = wave_reduce<true>(z);
    if (top == -INFINITY) top = 0.f;
    const float sum = wave_reduce<false>(exp_of(z - top, c2)), za = lane_of(z, label);
    if (lane == 0)
      a.row[row] = PrefRow{za == -INFINITY ? -(double)INFINITY : (double)za - (double)top - log_sum(sum), top, 1.f / sum};
  }
}

// The same where the row fits its threads' registers (E chunks each): all loads before any sum, two operations fewer an element.
// About 4100 counted rows of 32768 bf16 in 42 us (6.4 TB/s, part of it from the caches).
template <typename T, int NT, int E>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void pref_rows_held_kernel(PrefRows a) {
  constexpr int V = kVec<T>, PER = NT < 256 ? 256 / NT : 1;
  __shared__ float red[16];
  const int tid = threadIdx.x % NT;
  const int first = a.offsets[0], last = a.offsets[2 * a.pairs];
  const Base2 c2(1.0);
  for (int row = blockIdx.x * PER + wave_row<NT>(); row < a.rows; row += gridDim.x * PER) {
    const int label = a.label[row];
    if (tid == 0) a.coef[row] = 0.f;
    if (row < first || row >= last || (unsigned)label >= (unsigned)a.columns) continue;
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const Chunks<T> at(a.columns, z);
    u32x4 raw[E];
    load_row<T, NT, E>(z, tid, at, raw);
    const float za = (float)z[label];
    remove_past<T, NT, E>(tid, at, raw);
    const float top = max_of<T, NT, E>(raw, at, red), base = top == -INFINITY ? 0.f : top;
    forget<E>(raw);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (at.none(e * NT)) break;
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < V; j++) t += exp_of(element<T>(raw[e], j) - base, c2);
      sum += t;
      __builtin_amdgcn_sched_barrier(0);
    }
    const double total = row_sum<NT>(sum, red);
    if (tid == 0)
      a.row[row] = PrefRow{za == -INFINITY ? -(double)INFINITY : (double)za - (double)base - log_sum(total), base, (float)(1.0 / total)};
  }
}

// The same for longer rows, E chunks of each thread at a time relative to the running maximum. (Held by 1024 threads in 16
// chunks each, such a row has a CU to itself, whose loads and exponentials wait for each other: 297 us for 2430 rows of
// 100003 f16, against 116 here.) PARTS: few such rows in parts, with the label's logit in logp's place until pref_pairs_kernel
// joins them.
template <typename T, int NT, int E, bool PARTS>
__global__ __launch_bounds__(NT) void pref_rows_long_kernel(PrefRows a) {
  constexpr int V = kVec<T>;
  __shared__ float red[16];
  const int tid = threadIdx.x;
  const int first = a.offsets[0], last = a.offsets[2 * a.pairs];
  const Base2 c2(1.0);
  for (int id = blockIdx.x; id < a.rows * (PARTS ? a.split : 1); id += gridDim.x) {
    const int row = PARTS ? id / a.split : id, part = PARTS ? id - row * a.split : 0;
    const int begin = part * a.span, end = PARTS ? begin + a.span : INT_MAX;  // its chunks
    const int label = a.label[row];
    if (tid == 0 && part == 0) a.coef[row] = 0.f;
    if (row < first || row >= last || (unsigned)label >= (unsigned)a.columns) continue;
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    const Chunks<T> at(a.columns, z);
    Running run;
    for (int c0 = begin; c0 < end && !at.none(c0); c0 += NT * E) {
      u32x4 raw[E];
      load_row<T, NT, E>(z, tid, at, raw, c0);
      remove_past<T, NT, E>(tid, at, raw, c0);
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
    if (tid == 0) {
      const float za = (float)z[label];
      if constexpr (PARTS) {
        a.parts[id] = PrefPart{run.total, run.top, 0.f};
        if (part == 0) a.row[row].logp = (double)za;
        continue;
      }
      a.row[row] = PrefRow{za == -INFINITY ? -(double)INFINITY : (double)za - (double)run.top - log_sum(run.total), run.top,
                           (float)(1.0 / run.total)};
    }
  }
}

constexpr int PT = 512;  // threads of a pair's workgroup
// Preference rows cut into parts: 2 rows of 125123 f16 31 -> 14 us, 64 of 100003 bf16 32 -> 20, but 256 of them 37.5 -> 39.
constexpr int kPrefPartRows = 128;

// A row's results from its parts.
__device__ __forceinline__ PrefRow joined(const PrefRows& a, int row) {
  const PrefPart* q = a.parts + row * a.split;
  const Base2 c2(1.0);
  const double za = a.row[row].logp;
  float top = -INFINITY;
  for (int k = 0; k < a.split; k++) top = fmaxf(top, q[k].top);
  double sum = 0.0;
  for (int k = 0; k < a.split; k++) sum += q[k].sum * (double)(q[k].top == -INFINITY ? 0.f : exp_of(q[k].top - top, c2));
  return PrefRow{za == -(double)INFINITY ? za : za - (double)top - log_sum(sum), top, (float)(1.0 / sum)};
}

// One workgroup a pair: the sequences' sums in a fixed order, the loss, and the factor of each counted row's gradient. Bound by the
// latency of its dependent steps: 4.7 us at 6 pairs of 40 rows, 5.4 at 8 of 512.
__global__ __launch_bounds__(PT) void pref_pairs_kernel(PrefRows a) {
  __shared__ double sums[PT / 64][2];
  __shared__ int counts[PT / 64][2];
  const int tid = threadIdx.x, w = tid >> 6;
  for (int pair = blockIdx.x; pair < a.pairs; pair += gridDim.x) {
    int at[3];
    for (int k = 0; k < 3; k++) at[k] = min(max(a.offsets[2 * pair + k], 0), a.rows);
    double sum[2] = {0, 0};
    int count[2] = {0, 0};
#pragma unroll
    for (int q = 0; q < 2; q++) {
#pragma unroll 4
      for (int t = at[q] + tid; t < at[q + 1]; t += PT) {
        // (Every row's place is the workspace's own: read whether it counts or not, so that the loads run ahead.)
        const bool counted = (unsigned)a.label[t] < (unsigned)a.columns;
        if (counted && a.split > 1) a.row[t] = joined(a, t);
        const double lp = a.row[t].logp;
        sum[q] += counted ? lp : 0.0;
        count[q] += counted;
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        sum[q] += __shfl_xor(sum[q], o);
        count[q] += __shfl_xor(count[q], o);
      }
    }
    __syncthreads();
    if ((tid & 63) == 0)
      for (int q = 0; q < 2; q++) { sums[w][q] = sum[q]; counts[w][q] = count[q]; }
    __syncthreads();
    double part[2];
    for (int q = 0; q < 2; q++) {
      int n = 0;
      double total = 0.0;
      for (int k = 0; k < PT / 64; k++) {
        n += counts[k][q];
        total += sums[k][q];
      }
      part[q] = a.average ? 1.0 / max(n, 1) : 1.0;
      sum[q] = total * part[q];
    }
    const double h = a.beta * ((sum[0] - (double)a.ref_logp[2 * pair]) - (sum[1] - (double)a.ref_logp[2 * pair + 1]));
    const double wt = a.weight ? (double)a.weight[pair] : 1.0;
    // -log sigmoid(h) = log1p(e^-|h|) + max(-h, 0); the sigmoids from the same exponential.
    const double e = exp(-fabs(h)), soft = log1p(e), near = 1.0 / (1.0 + e), far = e / (1.0 + e);
    const double up = h >= 0 ? near : far, down = h >= 0 ? far : near;  // sigmoid(h), sigmoid(-h)
    if (tid == 0) {
      a.loss[pair] = (float)(wt * ((1 - a.smooth) * (soft + fmax(-h, 0.0)) + a.smooth * (soft + fmax(h, 0.0))));
      a.margin[pair] = (float)h;
      a.seq_logp[2 * pair] = (float)sum[0];
      a.seq_logp[2 * pair + 1] = (float)sum[1];
    }
    if (a.grad) {
      const double dh = wt * a.beta * (a.smooth * up - (1 - a.smooth) * down);
      for (int q = 0; q < 2; q++)
        for (int t = at[q] + tid; t < at[q + 1]; t += PT)
          if ((unsigned)a.label[t] < (unsigned)a.columns) a.coef[t] = (float)((q ? -dh : dh) * part[q]);
    }
  }
}

// The gradient of every row: first the sequences' rows, from the last to the first (what the sums read last is still in the
// caches), then the others, whose zeros would drive it out. Bound by memory, one read and one write: 8192 rows of 32768 bf16, half
// of them counted, in 123 us (6.5 TB/s), 5400 of 100003 f16 in 317 (4.9 TB/s).
template <typename T, int NT, int E>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void pref_grad_kernel(PrefRows a) {
  constexpr int V = kVec<T>, PER = NT < 256 ? 256 / NT : 1;
  const int tid = threadIdx.x % NT;
  // (Cut to the rows, so that each row comes once.)
  const int last = min(max(a.offsets[2 * a.pairs], 0), a.rows), first = min(max(a.offsets[0], 0), last);
  for (int id = blockIdx.x * PER + wave_row<NT>(); id < a.rows * a.split; id += gridDim.x * PER) {
    const int r = id / a.split, begin = (id - r * a.split) * a.span, end = a.split > 1 ? begin + a.span : INT_MAX;
    const int row = r < last - first ? last - 1 - r : r - (last - first) < first ? r - (last - first) : r;
    const int label = a.label[row];
    const bool counted = row >= first && row < last && (unsigned)label < (unsigned)a.columns;
    const T* z = (const T*)a.logits + (size_t)row * a.ld;
    T* g = (T*)a.grad + (size_t)row * a.ld_grad;
    const Chunks<T> at(a.columns, g);
    float hot = 0.f, f = 0.f, top = 0.f;
    if (counted) {
      hot = a.coef[row];
      top = a.row[row].top;
      f = -hot * a.row[row].inv_sum;
    }
    const int hot_chunk = counted ? at.of(label) : -1;
    for (int c0 = begin; c0 < end && !at.none(c0); c0 += NT * E) {
      u32x4 raw[E];
      if (counted) load_row<T, NT, E>(z, tid, at, raw, c0);
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (at.none(c0 + e * NT)) break;
        const int c = fresh(tid) + c0 + e * NT;
        float gf[V] = {};
        if (counted) {
#pragma unroll
          for (int j = 0; j < V; j++) gf[j] = __builtin_amdgcn_exp2f((element<T>(raw[e], j) - top) * 1.44269504088896340736f) * f;
          if (c == hot_chunk) {
            const int at_j = label - at.start(c);
#pragma unroll
            for (int j = 0; j < V; j++) gf[j] += j == at_j ? hot : 0.f;
          }
        }
        store_gradient<T>(g, c, at.whole(c0 + e * NT, NT), a.past, at, gf);
      }
    }
  }
}

// The same for rows shorter than a chunk.
template <typename T>
__global__ __launch_bounds__(256) void pref_grad_short_kernel(PrefRows a) {
  const int first = a.offsets[0], last = a.offsets[2 * a.pairs];
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)a.rows * a.columns; i += (long long)gridDim.x * 256) {
    const int row = (int)(i / a.columns), c = (int)(i % a.columns), label = a.label[row];
    float g = 0.f;
    if (row >= first && row < last && (unsigned)label < (unsigned)a.columns) {
      const float e = __builtin_amdgcn_exp2f(((float)((const T*)a.logits)[(size_t)row * a.ld + c] - a.row[row].top) * 1.44269504088896340736f);
      g = a.coef[row] * ((c == label ? 1.f : 0.f) - e * a.row[row].inv_sum);
    }
    ((T*)a.grad)[(size_t)row * a.ld_grad + c] = to_t<T>(g);
  }
}

template <typename T>
void pref_typed(PrefRows p, hipStream_t s) {
  const dim3 waves(row_grid(p.rows, 4)), groups(row_grid(p.rows, 1));
  const bool tiny = p.columns < kVec<T>;  // rows shorter than a chunk
  if (p.rows > 0) {
    const RowShape r = row_shape<T>(p.columns, p.logits, p.ld, p.rows);
    if (r.threads == 64 && r.each == 2) launch_k(pref_rows_held_kernel<T, 64, 2>, waves, 256, 0, s, p);
    else if (r.threads == 64) launch_k(pref_rows_held_kernel<T, 64, 8>, waves, 256, 0, s, p);
    else if (r.threads == 256) launch_k(pref_rows_held_kernel<T, 256, 8>, groups, 256, 0, s, p);
    else if (r.threads == 512) launch_k(pref_rows_held_kernel<T, 512, 8>, groups, 512, 0, s, p);
    else if (tiny) launch_k(pref_rows_short_kernel<T>, waves, 256, 0, s, p);
    else {
      if (p.rows <= kPrefPartRows) {
        const RowParts cut = row_parts<T>(p.rows, p.columns, 512 * 4);
        p.split = cut.split;
        p.span = cut.span;
      }
      if (p.split > 1) launch_k(pref_rows_long_kernel<T, 512, 4, true>, dim3(p.rows * p.split), 512, 0, s, p);
      else launch_k(pref_rows_long_kernel<T, 512, 4, false>, groups, 512, 0, s, p);
    }
  }
  if (p.pairs > 0) launch_k(pref_pairs_kernel, dim3(p.pairs < 65536 ? p.pairs : 65536), PT, 0, s, p);
  if (p.rows > 0 && p.grad) {
    if (tiny) launch_k(pref_grad_short_kernel<T>, dim3(row_grid(p.rows, 32)), 256, 0, s, p);
    else if (p.columns <= 512 * kVec<T>) launch_k(pref_grad_kernel<T, 64, 4>, waves, 256, 0, s, p);
    else if (p.columns <= 2048 * kVec<T>) launch_k(pref_grad_kernel<T, 256, 4>, groups, 256, 0, s, p);
    else launch_k(pref_grad_kernel<T, 512, 4>, dim3(row_grid(p.rows * p.split, 1)), 512, 0, s, p);
  }
}

}  // namespace

size_t policy_loss_workspace(int rows, int columns) {
  const int parts = most_parts(rows, columns);
  return parts > 1 ? (size_t)rows * parts * sizeof(PolicyPart) : 0;
}

void launch_policy_loss(const kg_policy_loss_args& a, hipStream_t s) {
  PolicyRows p;
  p.logits = a.logits; p.ld = a.ld;
  p.legal = a.legal; p.ld_legal = a.ld_legal;
  p.ref = a.ref_logits; p.ld_ref = a.ld_ref;
  p.grad = a.grad; p.ld_grad = a.ld_grad;
  p.action = a.action; p.old_logp = a.old_logp; p.advantage = a.advantage; p.weight = a.weight; p.ref_logp = a.ref_logp;
  p.loss = a.loss; p.logp = a.logp; p.kl = a.kl;
  p.rows = a.rows; p.columns = a.columns;
  p.past = gradient_past(a.rows, a.columns, a.type);
  p.scale = a.logit_scale;
  p.parts = (PolicyPart*)a.workspace;
  p.split = 1;
  p.span = 0;
  p.low = a.clip_low; p.high = a.clip_high;
  p.log_low = log1p(-a.clip_low); p.log_high = log1p(a.clip_high);
  p.kl_coef = (float)a.kl_coef;
  switch (a.type) {
    case PREC_F32: policy_typed<float>(p, s); break;
    case PREC_F16: policy_typed<f16>(p, s); break;
    default: policy_typed<bf16>(p, s); break;
  }
  KGX_CHECK_LAUNCH();
}

// The parts' place in the workspace, behind the rows' results and factors.
size_t pref_parts_at(int rows) { return ((size_t)rows * (sizeof(PrefRow) + sizeof(float)) + 15) / 16 * 16; }
size_t preference_loss_workspace(int rows) {
  if (rows < 1) return 0;
  const int parts = rows <= kPrefPartRows ? most_parts(rows, INT_MAX) : 1;
  return (pref_parts_at(rows) + (parts > 1 ? (size_t)rows * parts * sizeof(PrefPart) : 0) + 255) / 256 * 256;
}

void launch_preference_loss(const kg_preference_loss_args& a, hipStream_t s) {
  PrefRows p;
  p.logits = a.logits; p.ld = a.ld;
  p.grad = a.grad; p.ld_grad = a.ld_grad;
  p.label = a.label; p.offsets = a.offsets; p.ref_logp = a.ref_logp; p.weight = a.weight;
  p.row = (PrefRow*)a.workspace;
  p.coef = (float*)(p.row + a.rows);
  p.parts = (PrefPart*)((char*)a.workspace + pref_parts_at(a.rows));
  p.split = 1;
  p.span = 0;
  p.loss = a.loss; p.margin = a.margin; p.seq_logp = a.seq_logp;
  p.rows = a.rows; p.columns = a.columns; p.pairs = a.pairs; p.average = a.average;
  p.past = gradient_past(a.rows, a.columns, a.type);
  p.beta = a.beta; p.smooth = a.label_smoothing;
  switch (a.type) {
    case PREC_F32: pref_typed<float>(p, s); break;
    case PREC_F16: pref_typed<f16>(p, s); break;
    default: pref_typed<bf16>(p, s); break;
  }
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
