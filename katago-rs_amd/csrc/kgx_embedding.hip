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

struct SortArgs {
  const unsigned* keys;  // sorted by lower digits, with their places; the first pass reads the tokens themselves
  const int* places;
  unsigned* keys_out;
  int* places_out;
  int* counts;  // [blocks][2^bits]
  int count, vocab, blocks, each, shift, bits;  // each: tokens of a block, a multiple of ST
};

// Tokens outside the table are behind all others.
template <bool FIRST>
__device__ __forceinline__ unsigned key_of(const SortArgs& a, int i) {
  const unsigned k = a.keys[i];
  return FIRST && k >= (unsigned)a.vocab ? (unsigned)a.vocab : k;
}

template <bool FIRST>
__global__ __launch_bounds__(ST) void sort_count_kernel(SortArgs a) {
  __shared__ int n[1 << kDigit];
  const int digits = 1 << a.bits, tid = threadIdx.x;
  for (int b = blockIdx.x; b < a.blocks; b += gridDim.x) {
    for (int d = tid; d < digits; d += ST) n[d] = 0;
    __syncthreads();
    for (int r = 0; r < a.each; r += ST) {
      const long long i = (long long)b * a.each + r + tid;
      if (i < a.count) atomicAdd(&n[key_of<FIRST>(a, (int)i) >> a.shift & (digits - 1)], 1);
    }
    __syncthreads();
    for (int d = tid; d < digits; d += ST) a.counts[b * digits + d] = n[d];
    __syncthreads();
  }
}

template <bool FIRST>
__global__ __launch_bounds__(ST) void sort_move_kernel(SortArgs a) {
  constexpr int WAVES = ST / 64;
  __shared__ int to[WAVES][1 << kDigit];  // where a wave's next token of a digit goes
  __shared__ int total[1 << kDigit];
  const int digits = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, b = blockIdx.x;
  for (int d = tid; d < digits * WAVES; d += ST) to[d >> a.bits][d & (digits - 1)] = 0;
  int before = 0, all = 0;
  if (tid < digits)
    for (int k = 0; k < a.blocks; k++) {
      const int n = a.counts[k * digits + tid];
      before += k < b ? n : 0;
      all += n;
    }
  if (tid < digits) total[tid] = all;
  __syncthreads();
  // (The digits before this one, a doubling step at a time.)
  for (int o = 1; o < digits; o <<= 1) {
    const int v = tid < digits && tid >= o ? total[tid - o] : 0;
    __syncthreads();
    if (tid < digits) total[tid] += v;
    __syncthreads();
  }
  // A wave's tokens follow each other, and so do the waves.
  const int rounds = a.each / ST;
  const long long first = (long long)b * a.each + (long long)w * rounds * 64 + lane;
  for (int r = 0; r < rounds; r++)
    if (first + r * 64 < a.count) atomicAdd(&to[w][key_of<FIRST>(a, (int)(first + r * 64)) >> a.shift & (digits - 1)], 1);
  __syncthreads();
  if (tid < digits) {
    int at = total[tid] - all + before;
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
    const unsigned key = in ? key_of<FIRST>(a, (int)i) : 0u;
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
  int count, vocab, channels, ranges, each, accumulate;
  float scale;
};

template <typename T, typename G>
__device__ __forceinline__ void put(const SumArgs& a, unsigned key, int c, const float (&sum)[kVec<T>]) {
  G* g = (G*)a.grad + (size_t)key * a.ld_grad + c;
#pragma unroll
  for (int j = 0; j < kVec<T>; j++)
    if (c + j < a.channels) g[j] = to_t<G>(__builtin_fmaf(sum[j], a.scale, a.accumulate ? (float)g[j] : 0.f));
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

// A thread a column of 16 bytes of a range.
template <typename T, typename G>
__global__ __launch_bounds__(ET) void embedding_sums_kernel(SumArgs a, int chunks) {
  constexpr int V = kVec<T>;
  const long long all = (long long)a.ranges * chunks;
  for (long long id = (long long)blockIdx.x * ET + threadIdx.x; id < all; id += (long long)gridDim.x * ET) {
    const int range = (int)(id / chunks), c = (int)(id - (long long)range * chunks) * V;
    const int first = range * a.each, last = min(first + a.each, a.count);
    float sum[V] = {};
    unsigned key = a.keys[first];
    bool before = first > 0 && a.keys[first - 1] == key;
    auto leave = [&](int side) {
      float* p = a.parts + ((size_t)range * 2 + side) * a.channels + c;
      for (int j = 0; j < V; j++)
        if (c + j < a.channels) p[j] = sum[j];
    };
    for (int i = first; i < last && key < (unsigned)a.vocab; i++) {
      float f[V];
      load_vec<T>((const T*)a.dy + (size_t)a.places[i] * a.ld + c, a.channels - c, f);
#pragma unroll
      for (int j = 0; j < V; j++) sum[j] += f[j];
      const unsigned next = i + 1 < a.count ? a.keys[i + 1] : ~0u;
      if (next == key && i + 1 < last) continue;
      if (before) leave(0);
      else if (next == key) leave(1);
      else put<T, G>(a, key, c, sum);
#pragma unroll
      for (int j = 0; j < V; j++) sum[j] = 0.f;
      key = next;
      before = false;
    }
  }
}

// Runs over several ranges: a thread a column of the range that such a run begins in.
template <typename T, typename G>
__global__ __launch_bounds__(ET) void embedding_join_kernel(SumArgs a, int chunks) {
  constexpr int V = kVec<T>;
  const long long all = (long long)(a.ranges - 1) * chunks;
  for (long long id = (long long)blockIdx.x * ET + threadIdx.x; id < all; id += (long long)gridDim.x * ET) {
    const int range = (int)(id / chunks), c = (int)(id - (long long)range * chunks) * V;
    const int first = range * a.each, last = first + a.each;  // (one more range follows)
    const unsigned key = a.keys[last];
    if (key >= (unsigned)a.vocab || a.keys[last - 1] != key) continue;
    if (a.keys[first] == key && first > 0 && a.keys[first - 1] == key) continue;  // begins before
    const int ends = (lower_bound(a.keys, a.count, key + 1) - 1) / a.each;        // the range of its last token
    double sum[V] = {};
    for (int r = range; r <= ends; r++) {
      const float* p = a.parts + ((size_t)r * 2 + (r == range)) * a.channels + c;
#pragma unroll
      for (int j = 0; j < V; j++) sum[j] += c + j < a.channels ? (double)p[j] : 0.0;
    }
    float f[V];
#pragma unroll
    for (int j = 0; j < V; j++) f[j] = (float)sum[j];
    put<T, G>(a, key, c, f);
  }
}

// Rows that no token names.
template <typename G>
__global__ __launch_bounds__(ET) void embedding_fill_kernel(SumArgs a) {
  for (int row = blockIdx.x; row < a.vocab; row += gridDim.x) {
    const int at = lower_bound(a.keys, a.count, (unsigned)row);
    if (at < a.count && a.keys[at] == (unsigned)row) continue;
    G* g = (G*)a.grad + (size_t)row * a.ld_grad;
    for (int c = threadIdx.x; c < a.channels; c += ET) g[c] = to_t<G>(0.f);
  }
}

// How the tokens are sorted and cut, and where their parts of the workspace lie.
struct Plan {
  int passes, bits, blocks, each_block, each, ranges;
  size_t keys, places, counts, parts, bytes;
};
Plan plan_of(int count, int vocab, int channels) {
  Plan p;
  const int bits = 32 - __builtin_clz((unsigned)vocab);  // of the keys 0 ... vocab
  p.passes = (bits + kDigit - 1) / kDigit;
  p.bits = (bits + p.passes - 1) / p.passes;
  const long long rounds = ((long long)count + (long long)ST * kMostBlocks - 1) / ((long long)ST * kMostBlocks);
  p.each_block = (int)(rounds * ST);
  p.blocks = (int)(((long long)count + p.each_block - 1) / p.each_block);
  p.each = (int)std::max(((long long)count + 2047) / 2048, 16ll);
  p.ranges = (int)(((long long)count + p.each - 1) / p.each);
  const auto room = [&](size_t n) {
    const size_t at = p.bytes;
    p.bytes += (n + 255) / 256 * 256;
    return at;
  };
  p.bytes = 0;
  p.keys = room((size_t)count * 8);
  p.places = room((size_t)count * 8);
  p.counts = room((size_t)p.blocks * (4 << p.bits));
  p.parts = room((size_t)p.ranges * 2 * channels * 4);
  return p;
}

inline int grid_of(long long threads) { return (int)std::min((threads + ET - 1) / ET, 1ll << 20); }

template <typename T, typename G>
void backward_typed(const SumArgs& p, hipStream_t s) {
  const int chunks = (p.channels + kVec<T> - 1) / kVec<T>;
  if (p.count) launch_k(embedding_sums_kernel<T, G>, dim3(grid_of((long long)p.ranges * chunks)), ET, 0, s, p, chunks);
  if (p.ranges > 1) launch_k(embedding_join_kernel<T, G>, dim3(grid_of((long long)(p.ranges - 1) * chunks)), ET, 0, s, p, chunks);
  if (!p.accumulate) launch_k(embedding_fill_kernel<G>, dim3(std::min(p.vocab, 1 << 20)), ET, 0, s, p);
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
    char* w = (char*)a.workspace;
    unsigned* keys = (unsigned*)(w + plan.keys);
    int* places = (int*)(w + plan.places);
    SortArgs t;
    t.keys = (const unsigned*)a.tokens;
    t.places = nullptr;
    t.counts = (int*)(w + plan.counts);
    t.count = a.count; t.vocab = a.vocab; t.blocks = plan.blocks; t.each = plan.each_block; t.bits = plan.bits;
    for (int k = 0; k < plan.passes; k++) {
      t.shift = k * plan.bits;
      t.keys_out = keys + (size_t)(k & 1) * a.count;
      t.places_out = places + (size_t)(k & 1) * a.count;
      if (k == 0) {
        launch_k(sort_count_kernel<true>, dim3(t.blocks), ST, 0, s, t);
        launch_k(sort_move_kernel<true>, dim3(t.blocks), ST, 0, s, t);
      } else {
        launch_k(sort_count_kernel<false>, dim3(t.blocks), ST, 0, s, t);
        launch_k(sort_move_kernel<false>, dim3(t.blocks), ST, 0, s, t);
      }
      t.keys = t.keys_out;
      t.places = t.places_out;
    }
    p.keys = t.keys;
    p.places = t.places;
    p.parts = (float*)(w + plan.parts);
    p.ranges = plan.ranges;
    p.each = plan.each;
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
