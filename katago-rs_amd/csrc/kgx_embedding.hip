// The rows of a table that tokens name, scaled, and the table's gradient (kg_embedding, kg_embedding_backward).
//
// The gradient of a row is the sum of its tokens' gradients, in the order of the tokens whatever runs first: the tokens are sorted
// with their places (stable, by digits of at most 9 bits; counts are whole numbers, so that their atomics have no order), and the sorted
// places are cut into ranges of equal length, so that a token that comes often is no longer than many that come once. A range sums
// its runs of one token each; a run that reaches over its range's ends leaves its sum to a second launch, which adds such sums up.
// Rows that no token names are filled with 0 by other workgroups of the first.
#include <algorithm>

#include "kgx_device.h"
#include "kgx_learn.h"
#include "kgx_vec.h"

namespace kgx {

namespace {

constexpr int ET = 256;       // threads of a workgroup
constexpr int ST = 1024;      // of the sort's
constexpr int kDigit = 9;     // bits of a digit, at most
constexpr int kMostBlocks = 64;  // of tokens, in the sort
constexpr int FR = 16;        // rows that a wave looks for at once

template <typename T>
__global__ __launch_bounds__(ET) void embedding_kernel(const int* tokens, const T* table, T* y, long long ld, long long ld_y, int count,
                                                       int vocab, int channels, int chunks, float scale) {
  constexpr int V = kVec<T>;
  const long long all = (long long)count * chunks;
  for (long long id = (long long)blockIdx.x * ET + threadIdx.x; id < all; id += (long long)gridDim.x * ET) {
    const int i = (int)(id / chunks), c = (int)(id - (long long)i * chunks) * V, token = tokens[i];
    float f[V] = {};
    if ((unsigned)token < (unsigned)vocab) {
      load_vec<T>(table + (size_t)token * ld + c, channels - c, f);
#pragma unroll
      for (int j = 0; j < V; j++) f[j] *= scale;
    }
    store_vec<T>(y + (size_t)i * ld_y + c, channels - c, f);
  }
}

// ---- The sort. ----

// Tokens outside the table are behind all others.
__device__ __forceinline__ unsigned key_of(int token, int vocab) { return min((unsigned)token, (unsigned)vocab); }

// Few tokens: each one's place is the number of tokens before it, counted. RI tokens a workgroup, whose threads share the tokens
// that they are compared with, 64 ways: 5003 tokens in 5 us, where two launches for each digit take 20.
constexpr int kRanked = 8192, RI = 16;
__global__ __launch_bounds__(ST) void sort_rank_kernel(const int* __restrict__ tokens, unsigned* __restrict__ keys, int* __restrict__ places,
                                                       int count, int vocab) {
  __shared__ __align__(16) unsigned all[kRanked];
  __shared__ int part[ST / 64][RI];
  const int tid = threadIdx.x, w = tid >> 6, item = tid & (RI - 1), share = (w << 2) | (tid & 63) / RI;
  const int room = (count + 255) / 256 * 256;  // (64 shares of whole fours)
  for (int i = tid; i < room; i += ST) all[i] = i < count ? key_of(tokens[i], vocab) : ~0u;
  __syncthreads();
  const int i = blockIdx.x * RI + item;
  const unsigned key = all[min(i, room - 1)];
  // A token before this one counts where its key is no larger, one behind where it is less: the shares cross from the ones to the others
  // at i.
  int n = 0;
  for (int j = share * 4; j < room; j += 256) {
    const uint4 k = *(const uint4*)(all + j);
    n += (k.x < key + (j < i)) + (k.y < key + (j + 1 < i)) + (k.z < key + (j + 2 < i)) + (k.w < key + (j + 3 < i));
  }
  for (int o = RI; o < 64; o <<= 1) n += __shfl_xor(n, o);
  if ((tid & 63) < RI) part[w][item] = n;
  __syncthreads();
  if (tid < RI && i < count) {
    int at = 0;
    for (int k = 0; k < ST / 64; k++) at += part[k][tid];
    keys[at] = key;
    places[at] = i;
  }
}

// More: by digits from the lowest, two launches for the first and one for each other: a launch that moves the tokens by a digit counts
// the next digit at their new places.
struct SortArgs {
  const int* tokens;
  const unsigned* keys;  // sorted by lower digits, with their places; the first pass reads the tokens themselves
  const int* places;
  unsigned* keys_out;
  int* places_out;
  int *counts, *next_counts;  // [blocks][2^bits] of this digit and, but for the last, the next one
  int count, vocab, blocks, each, shift, bits, rest;  // each: tokens of a block, a multiple of ST; rest: counts behind these, to be cleared
};

__global__ __launch_bounds__(ST) void sort_count_kernel(SortArgs a) {
  __shared__ int n[1 << kDigit];
  const int digits = 1 << a.bits, tid = threadIdx.x, b = blockIdx.x;
  for (int d = tid; d < digits; d += ST) n[d] = 0;
  for (int k = b * ST + tid; k < a.rest; k += a.blocks * ST) a.next_counts[k] = 0;
  __syncthreads();
  for (int r = 0; r < a.each; r += ST) {
    const long long i = (long long)b * a.each + r + tid;
    if (i < a.count) atomicAdd(&n[key_of(a.tokens[i], a.vocab) & (digits - 1)], 1);
  }
  __syncthreads();
  for (int d = tid; d < digits; d += ST) a.counts[b * digits + d] = n[d];
}

template <bool FIRST, bool LAST>
__global__ __launch_bounds__(ST) void sort_move_kernel(SortArgs a) {
  constexpr int WAVES = ST / 64;
  __shared__ int to[WAVES][1 << kDigit];  // where a wave's next token of a digit goes
  __shared__ int sums[WAVES];
  const int digits = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, b = blockIdx.x;
  const auto key_at = [&](long long i) { return FIRST ? key_of(a.tokens[i], a.vocab) : a.keys[i]; };
  for (int d = tid; d < digits * WAVES; d += ST) to[d >> a.bits][d & (digits - 1)] = 0;
  int before = 0, all = 0;
  if (tid < digits) {
#pragma unroll 16
    for (int k = 0; k < a.blocks; k++) {
      const int n = a.counts[k * digits + tid];
      before += k < b ? n : 0;
      all += n;
    }
  }
  // The tokens of lower digits: within a wave, then over the waves.
  int upto = all;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(upto, o);
    upto += lane >= o ? v : 0;
  }
  if (lane == 63) sums[w] = upto;
  __syncthreads();
  for (int k = 0; k < w; k++) upto += sums[k];
  // A wave's tokens follow each other, and so do the waves.
  const int rounds = a.each / ST;
  const long long first = (long long)b * a.each + (long long)w * rounds * 64 + lane;
  for (int r = 0; r < rounds; r++)
    if (first + r * 64 < a.count) atomicAdd(&to[w][key_at(first + r * 64) >> a.shift & (digits - 1)], 1);
  __syncthreads();
  if (tid < digits) {
    int at = upto - all + before;
    for (int k = 0; k < WAVES; k++) {
      const int n = to[k][tid];
      to[k][tid] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int r = 0; r < rounds; r++) {
    const long long i = first + r * 64;
    const bool in = i < a.count;
    const unsigned key = in ? key_at(i) : 0u;
    const unsigned d = key >> a.shift & (digits - 1);
    unsigned long long same = __ballot(in);
    for (int k = 0; k < a.bits; k++) {
      const unsigned long long set = __ballot(d >> k & 1);
      same &= d >> k & 1 ? set : ~set;
    }
    if (in) {
      const int at = to[w][d] + __popcll(same & ((1ull << lane) - 1));
      a.keys_out[at] = key;
      a.places_out[at] = FIRST ? (int)i : a.places[i];
      if (same >> lane == 1) to[w][d] = at + 1;  // (the last of its digit; the reads above came before, in one wave's order)
      if (!LAST) atomicAdd(&a.next_counts[at / a.each * digits + (key >> (a.shift + a.bits) & (digits - 1))], 1);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- The sums. ----

struct SumArgs {
  const unsigned* keys;
  const int* places;
  const void* dy;
  void* grad;
  float* parts;  // [ranges][2][channels]: the sum of a run from before the range, and of one that goes on behind it
  long long ld, ld_grad;
  int count, vocab, channels, ranges, each, slabs, sum_groups, accumulate;  // slabs: of a row's columns; sum_groups: workgroups that sum
  float scale;
};

// N values at p, of which `left` are the row's.
template <typename G, int N>
__device__ __forceinline__ void put(G* p, int left, const float (&sum)[N], float scale, int accumulate) {
  constexpr int V = N < kVec<G> ? N : kVec<G>;
#pragma unroll
  for (int h = 0; h < N; h += V) {
    if constexpr (V == kVec<G>) {
      float f[V] = {};
      if (accumulate) load_vec<G>(p + h, left - h, f);
#pragma unroll
      for (int j = 0; j < V; j++) f[j] = __builtin_fmaf(sum[h + j], scale, f[j]);
      store_vec<G>(p + h, left - h, f);
    } else {
#pragma unroll
      for (int j = 0; j < V; j++)
        if (h + j < left) p[h + j] = to_t<G>(__builtin_fmaf(sum[h + j], scale, accumulate ? (float)p[h + j] : 0.f));
    }
  }
}

// The first sorted place whose key is at least `key`.
__device__ __forceinline__ int lower_bound(const unsigned* keys, int count, unsigned key) {
  int lo = 0, n = count;
  while (n > 0) {
    const int half = n >> 1;
    if (keys[lo + half] < key) {
      lo += half + 1;
      n -= half + 1;
    } else {
      n = half;
    }
  }
  return lo;
}

// Rows that no token names: a wave looks for FR at once and fills them in turn.
template <typename G>
__device__ __forceinline__ void fill_rows(const SumArgs& a, int wave, int waves) {
  const int lane = threadIdx.x & 63;
  for (long long row = (long long)wave * FR; row < a.vocab; row += (long long)waves * FR) {
    bool none = false;
    if (lane < FR && row + lane < a.vocab) {
      const unsigned key = (unsigned)row + lane;
      const int at = lower_bound(a.keys, a.count, key);
      none = at >= a.count || a.keys[at] != key;
    }
    const float zeros[kVec<G>] = {};
    for (unsigned long long left = __ballot(none); left; left &= left - 1) {
      G* g = (G*)a.grad + (size_t)(row + __ffsll((unsigned long long)left) - 1) * a.ld_grad;
      for (int c = lane * kVec<G>; c < a.channels; c += 64 * kVec<G>) store_vec<G>(g + c, a.channels - c, zeros);
    }
  }
}

// L lanes take a slab of L columns of 16 bytes over a range, eight tokens' loads at a time. The workgroups behind fill.
template <typename T, typename G, int L>
__global__ __launch_bounds__(ET) void embedding_sums_kernel(SumArgs a) {
  constexpr int V = kVec<T>, AT_ONCE = 8;
  if ((int)blockIdx.x >= a.sum_groups) {
    fill_rows<G>(a, __builtin_amdgcn_readfirstlane((blockIdx.x - a.sum_groups) * (ET / 64) + (threadIdx.x >> 6)),
                 (gridDim.x - a.sum_groups) * (ET / 64));
    return;
  }
  const int lane = threadIdx.x % L;
  const auto from = [&](int v, int t) {  // of the lane that has token t
    if constexpr (L == 64) return __builtin_amdgcn_readlane(v, t);
    else return __shfl(v, t, L);
  };
  int unit = blockIdx.x * (ET / L) + threadIdx.x / L;
  if (L == 64) unit = __builtin_amdgcn_readfirstlane(unit);
  const int range = unit / a.slabs, c = ((unit - range * a.slabs) * L + lane) * V;
  if (range >= a.ranges) return;
  const int left = max(a.channels - c, 0), first = range * a.each, last = min(first + a.each, a.count);
  float sum[V] = {};
  int run = (int)a.keys[first];
  bool before = first > 0 && (int)a.keys[first - 1] == run;
  const int next = last < a.count ? (int)a.keys[last] : -1;
  const auto end_run = [&](bool after) {
    if (before || after) {
      float* p = a.parts + ((size_t)range * 2 + (before ? 0 : 1)) * a.channels + c;
#pragma unroll
      for (int h = 0; h < V; h += 4) {
        const float f[4] = {sum[h], sum[h + 1], sum[h + 2], sum[h + 3]};
        store_vec<float>(p + h, left - h, f);
      }
    } else {
      put<G, V>((G*)a.grad + (size_t)run * a.ld_grad + c, left, sum, a.scale, a.accumulate);
    }
  };
  for (int i0 = first; i0 < last; i0 += L) {
    int key = a.vocab, place = 0;
    if (i0 + lane < last) {
      key = (int)a.keys[i0 + lane];
      place = a.places[i0 + lane];
    }
#pragma unroll 1
    for (int u = 0; u < L; u += AT_ONCE) {
      if (i0 + u >= last || from(key, u) >= a.vocab) break;
      typename RowVec<T>::type raw[AT_ONCE];
      const bool whole = left >= V;
#pragma unroll
      for (int t = 0; t < AT_ONCE; t++) {
        const int k = from(key, u + t), at = from(place, u + t);  // (of lanes that a branch on `whole` would switch off)
        if (k < a.vocab && whole) raw[t] = *(const typename RowVec<T>::type*)((const T*)a.dy + (size_t)at * a.ld + c);
      }
#pragma unroll
      for (int t = 0; t < AT_ONCE; t++) {
        const int k = from(key, u + t), at = from(place, u + t);
        if (k >= a.vocab) continue;
        if (k != run) {
          end_run(false);
#pragma unroll
          for (int j = 0; j < V; j++) sum[j] = 0.f;
          run = k;
          before = false;
        }
        if (whole) {
#pragma unroll
          for (int j = 0; j < V; j++) sum[j] += widen1<T>(raw[t], j);
        } else {
          const T* p = (const T*)a.dy + (size_t)at * a.ld + c;
#pragma unroll
          for (int j = 0; j < V; j++) sum[j] += j < left ? (float)p[j] : 0.f;
        }
      }
    }
  }
  if (run < a.vocab) end_run(next == run);
}

// Runs over several ranges: a workgroup for 256 channels of each range that such a run begins in, its waves for the ranges in turn.
constexpr int JT = 512;
template <typename G>
__global__ __launch_bounds__(JT) void embedding_join_kernel(SumArgs a, int slabs) {
  __shared__ double joined[JT / 64][64][4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const long long all = (long long)(a.ranges - 1) * slabs;
  for (long long id = blockIdx.x; id < all; id += gridDim.x) {
    const int range = (int)(id / slabs), c = (int)(id - (long long)range * slabs) * 256 + lane * 4;
    const int first = range * a.each, last = first + a.each;  // (one more range follows)
    const unsigned key = a.keys[last];
    if (key >= (unsigned)a.vocab || a.keys[last - 1] != key) continue;
    if (a.keys[first] == key && first > 0 && a.keys[first - 1] == key) continue;  // begins before
    const int ends = (lower_bound(a.keys, a.count, key + 1) - 1) / a.each;        // the range of its last token
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
    for (int r = range + w; r <= ends; r += JT / 64) {
      float f[4];
      load_vec<float>(a.parts + ((size_t)r * 2 + (r == range)) * a.channels + c, max(a.channels - c, 0), f);
#pragma unroll
      for (int j = 0; j < 4; j++) sum[j] += (double)f[j];
    }
#pragma unroll
    for (int j = 0; j < 4; j++) joined[w][lane][j] = sum[j];
    __syncthreads();
    if (w == 0) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        double t = 0.0;
        for (int k = 0; k < JT / 64; k++) t += joined[k][lane][j];
        f[j] = (float)t;
      }
      put<G, 4>((G*)a.grad + (size_t)key * a.ld_grad + c, max(a.channels - c, 0), f, a.scale, a.accumulate);
    }
    __syncthreads();
  }
}

// How the tokens are sorted and cut, and where their parts of the workspace lie.
struct Plan {
  int passes, bits, blocks, each_block, each, ranges;  // passes: 0 where the tokens are ranked
  size_t keys, places, counts, parts, bytes;
};
// (Ranges of as many tokens as leave some 2048 waves with a row's columns; a run's sum of more than 256 is cut.)
Plan plan_of(int count, int vocab, int channels) {
  Plan p = {};
  if (count > kRanked) {
    const int bits = 32 - __builtin_clz((unsigned)vocab);  // of the keys 0 ... vocab
    p.passes = (bits + kDigit - 1) / kDigit;
    p.bits = (bits + p.passes - 1) / p.passes;
    const long long rounds = ((long long)count + (long long)ST * kMostBlocks - 1) / ((long long)ST * kMostBlocks);
    p.each_block = (int)(rounds * ST);
    p.blocks = (int)(((long long)count + p.each_block - 1) / p.each_block);
  }
  const long long slabs = ((long long)channels + 511) / 512;
  p.each = (int)std::min(std::max((long long)count * std::min(slabs, 64ll) / 2048, 8ll) / 8 * 8, 256ll);
  p.ranges = (int)(((long long)count + p.each - 1) / p.each);
  const auto room = [&](size_t n) {
    const size_t at = p.bytes;
    p.bytes += (n + 255) / 256 * 256;
    return at;
  };
  const size_t copies = p.passes > 1 ? 2 : 1;
  p.keys = room(copies * count * 4);
  p.places = room(copies * count * 4);
  p.counts = room((size_t)p.passes * p.blocks * (4 << p.bits));
  p.parts = room((size_t)p.ranges * 2 * channels * 4);
  return p;
}

inline int grid_of(long long threads) { return (int)std::min((threads + ET - 1) / ET, 1ll << 20); }

void sort_tokens(const kg_embedding_args& a, const Plan& plan, SumArgs& p, hipStream_t s) {
  char* w = (char*)a.workspace;
  unsigned* keys = (unsigned*)(w + plan.keys);
  int* places = (int*)(w + plan.places);
  int* counts = (int*)(w + plan.counts);
  p.keys = keys;
  p.places = places;
  if (!plan.passes) {
    launch_k(sort_rank_kernel, dim3((a.count + RI - 1) / RI), ST, 0, s, a.tokens, keys, places, a.count, a.vocab);
    return;
  }
  const int of_pass = plan.blocks << plan.bits;
  SortArgs t = {};
  t.tokens = a.tokens;
  t.count = a.count; t.vocab = a.vocab; t.blocks = plan.blocks; t.each = plan.each_block; t.bits = plan.bits;
  for (int k = 0; k < plan.passes; k++) {
    const dim3 grid(t.blocks);
    const bool last = k == plan.passes - 1;
    t.shift = k * plan.bits;
    t.keys_out = keys + (size_t)(k & 1) * a.count;
    t.places_out = places + (size_t)(k & 1) * a.count;
    t.counts = counts + (size_t)k * of_pass;
    t.next_counts = t.counts + of_pass;
    if (k == 0) {
      t.rest = (plan.passes - 1) * of_pass;
      launch_k(sort_count_kernel, grid, ST, 0, s, t);
      if (last) launch_k(sort_move_kernel<true, true>, grid, ST, 0, s, t);
      else launch_k(sort_move_kernel<true, false>, grid, ST, 0, s, t);
    } else if (last) {
      launch_k(sort_move_kernel<false, true>, grid, ST, 0, s, t);
    } else {
      launch_k(sort_move_kernel<false, false>, grid, ST, 0, s, t);
    }
    p.keys = t.keys = t.keys_out;
    p.places = t.places = t.places_out;
  }
}

template <typename T, typename G, int L>
void sums(SumArgs p, hipStream_t s) {
  const int chunks = (p.channels + kVec<T> - 1) / kVec<T>;
  p.slabs = (chunks + L - 1) / L;
  p.sum_groups = (int)(((long long)p.ranges * p.slabs + ET / L - 1) / (ET / L));
  const int fill = p.accumulate ? 0 : (int)std::min(((long long)p.vocab + FR * ET / 64 - 1) / (FR * ET / 64), 8192ll);
  launch_k(embedding_sums_kernel<T, G, L>, dim3(p.sum_groups + fill), ET, 0, s, p);
  if (p.ranges > 1) {
    const int slabs = (p.channels + 255) / 256;
    launch_k(embedding_join_kernel<G>, dim3((int)std::min((long long)(p.ranges - 1) * slabs, 1ll << 20)), JT, 0, s, p, slabs);
  }
}
template <typename T, typename G>
void backward_typed(const SumArgs& p, hipStream_t s) {
  const int chunks = (p.channels + kVec<T> - 1) / kVec<T>;
  if (chunks <= 16) sums<T, G, 16>(p, s);
  else if (chunks <= 32) sums<T, G, 32>(p, s);
  else sums<T, G, 64>(p, s);
}

}  // namespace

size_t embedding_backward_workspace(int count, int vocab, int channels) { return count < 1 ? 0 : plan_of(count, vocab, channels).bytes; }

void launch_embedding(const kg_embedding_args& a, hipStream_t s) {
  const float scale = (float)a.scale;
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    const int chunks = (a.channels + kVec<T> - 1) / kVec<T>;
    launch_k(embedding_kernel<T>, dim3(grid_of((long long)a.count * chunks)), ET, 0, s, a.tokens, (const T*)a.table, (T*)a.y, a.ld_table,
             a.ld_y, a.count, a.vocab, a.channels, chunks, scale);
  };
  switch (a.type) {
    case PREC_F32: go(0.f); break;
    case PREC_F16: go((f16)0.f); break;
    default: go((bf16)0.f); break;
  }
  KGX_CHECK_LAUNCH();
}

void launch_embedding_backward(const kg_embedding_args& a, hipStream_t s) {
  SumArgs p = {};
  p.dy = a.dy; p.ld = a.ld_dy;
  p.grad = a.grad; p.ld_grad = a.ld_grad;
  p.count = a.count; p.vocab = a.vocab; p.channels = a.channels; p.accumulate = a.accumulate != 0;
  p.scale = (float)a.scale;
  if (a.count) {
    const Plan plan = plan_of(a.count, a.vocab, a.channels);
    p.parts = (float*)((char*)a.workspace + plan.parts);
    p.ranges = plan.ranges;
    p.each = plan.each;
    sort_tokens(a, plan, p, s);
  }
  if (a.grad_type == a.type) {
    switch (a.type) {
      case PREC_F32: backward_typed<float, float>(p, s); break;
      case PREC_F16: backward_typed<f16, f16>(p, s); break;
      default: backward_typed<bf16, bf16>(p, s); break;
    }
  } else if (a.type == PREC_F16) {
    backward_typed<f16, float>(p, s);
  } else {
    backward_typed<bf16, float>(p, s);
  }
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
