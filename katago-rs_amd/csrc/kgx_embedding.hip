// The rows of a table that tokens name, scaled, and the table's gradient (kg_embedding, kg_embedding_backward).
//
// The gradient of a row is the sum of its tokens' gradients, in an order that the tokens alone decide: they are sorted with their places
// (stable, by counting where there are few, else by digits of at most 9 bits; counts are whole numbers, so that their atomics have no
// order), and the sorted places are cut into ranges of equal length, so that a token that comes often takes no longer than many that come
// once. A workgroup sums the runs of one token each in a range, in shares; a run that reaches over its range's ends leaves its sum to a
// last launch, which adds such sums up. Rows that no token names are 0: filled beside the sums, or all of them beside the sort. Few tokens
// of a small table take one launch instead (embedding_few_kernel).
#include <algorithm>

#include "kgx_device.h"
#include "kgx_learn.h"
#include "kgx_rows.h"

namespace kgx {

namespace {

constexpr int ET = 256;       // threads of a workgroup
constexpr int ST = 1024;      // of the sort's
constexpr int kDigit = 9;     // bits of a digit, at most
constexpr int kMostBlocks = 256;  // of tokens, in the sort
constexpr long long kFewColumns = 1 << 20;  // two threads for each that the card holds
constexpr int FR = 16;        // rows that a wave looks for at once

// Rows go by vectors of V elements: 16 bytes, the last of a row overlapping the one before (both have the same values of what they share),
// or single elements where the row is shorter.
template <typename T, int V>
__device__ __forceinline__ void load_columns(const T* p, float (&f)[V]) {
  if constexpr (V == 1) f[0] = (float)p[0];
  else load_vec<T>(p, V, f);
}

// A thread a vector of EACH rows, whose loads are under way together.
template <typename T, int V, int EACH>
__global__ __launch_bounds__(ET) void embedding_kernel(const int* tokens, const T* table, T* y, long long ld, long long ld_y, int count,
                                                       int vocab, int channels, int chunks, float scale, int past) {
  const int groups = (count + EACH - 1) / EACH;
  const long long all = (long long)groups * chunks;
  for (long long id = (long long)blockIdx.x * ET + threadIdx.x; id < all; id += (long long)gridDim.x * ET) {
    const int group = (int)(id / chunks), c = min((int)(id - (long long)group * chunks) * V, channels - V), i0 = group * EACH;
    float f[EACH][V] = {};
    int token[EACH];
#pragma unroll
    for (int k = 0; k < EACH; k++) token[k] = i0 + k < count ? tokens[i0 + k] : -1;
#pragma unroll
    for (int k = 0; k < EACH; k++)
      if ((unsigned)token[k] < (unsigned)vocab) load_columns<T, V>(table + (size_t)token[k] * ld + c, f[k]);
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      if (i0 + k >= count) break;
#pragma unroll
      for (int j = 0; j < V; j++) f[k][j] *= scale;
      T* to = y + (size_t)(i0 + k) * ld_y + c;
      if constexpr (V == 1) *to = to_t<T>(f[k][0]);
      else if (past) store_past<T>(to, f[k]);
      else store_vec<T>(to, V, f[k]);
    }
  }
}

// ---- The sort. ----

// Tokens outside the table are behind all others.
__device__ __forceinline__ unsigned key_of(int token, int vocab) { return min((unsigned)token, (unsigned)vocab); }

// 0 in rows of the table by workgroups behind those that sort, whose launches leave memory idle. In every row, which the sums then write over,
// where few are named or the table is small (5003 tokens of 100003 rows of 512 f16: 28 us, 32 with the others looked for and filled
// beside the sums). Or in those that no token names, by marks that the first launch leaves: a row's is the place of any of its tokens, so that
// what was in the marks' memory before is no mark unless it happens to be true (20000 tokens of 50257 rows of 1024 floats 62 -> 58 us
// against filling beside the sums, 65536 of 200000 of 512 129 -> 120).
struct FillArgs {
  void* grad;
  long long ld;     // bytes
  long long bytes;
  const int *tokens, *marks;  // marks: [vocab], or NULL: every row
  int count, first, rows, groups;  // this launch's rows; groups: workgroups that sort
};
constexpr int kMarked = 8;  // rows whose marks a wave reads at once
__device__ __forceinline__ void fill_row(const FillArgs& f, int row) {
  char* p = (char*)f.grad + (size_t)row * f.ld;
  for (long long c = (threadIdx.x & 63) * 16; c < f.bytes; c += 1024) {
    if (c + 16 <= f.bytes) *(u32x4_any2*)(p + c) = u32x4{0, 0, 0, 0};
    else for (long long k = c; k < f.bytes; k += 2) *(unsigned short*)(p + k) = 0;
  }
}
__device__ __forceinline__ bool fills(const FillArgs& f) {
  if ((int)blockIdx.x < f.groups) return false;
  const int lane = threadIdx.x & 63, end = f.first + f.rows, waves = (gridDim.x - f.groups) * (ST / 64);
  const int wave = __builtin_amdgcn_readfirstlane((blockIdx.x - f.groups) * (ST / 64) + (threadIdx.x >> 6));
  if (!f.marks) {
    for (int row = f.first + wave; row < end; row += waves) fill_row(f, row);
    return true;
  }
  for (long long row = f.first + (long long)wave * kMarked; row < end; row += (long long)waves * kMarked) {
    bool none = false;
    if (lane < kMarked && row + lane < end) {
      const int at = f.marks[row + lane];
      none = (unsigned)at >= (unsigned)f.count || f.tokens[at] != (int)row + lane;
    }
    for (unsigned long long left = __ballot(none); left; left &= left - 1) fill_row(f, (int)row + __ffsll(left) - 1);
  }
  return true;
}

// Few tokens: each one's place is the number of tokens before it, counted. RI tokens a workgroup, whose threads share the tokens
// that they are compared with, 64 ways: 5003 tokens in 8 us, where two launches for each of two digits take 22.
constexpr int kRanked = 8192, RI = 16;
__global__ __launch_bounds__(ST) void sort_rank_kernel(const int* __restrict__ tokens, unsigned* __restrict__ keys, int* __restrict__ places,
                                                       int count, int vocab, FillArgs fill) {
  if (fills(fill)) return;
  __shared__ __align__(16) unsigned all[kRanked];
  __shared__ int part[ST / 64][RI];
  const int tid = threadIdx.x, w = tid >> 6, item = tid & (RI - 1), share = (w << 2) | (tid & 63) / RI;
  const int room = (count + 255) / 256 * 256;  // (64 shares of whole fours)
  for (int i = tid; i < room; i += ST) all[i] = i < count ? key_of(tokens[i], vocab) : ~0u;
  __syncthreads();
  const int i = blockIdx.x * RI + item;
  const unsigned key = all[min(i, room - 1)];
  // A token before this one counts where its key is no larger, one behind where it is less. Those of the workgroup's own RI are both.
  const int i0 = blockIdx.x * RI;
  int n = 0;
  for (int j = share * 4; j < room; j += 256) {
    const uint4 k = *(const uint4*)(all + j);
    const unsigned limit = key + (j < i0);
    n += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
    if (j >= i0 && j < i0 + RI) n += (k.x == key && j < i) + (k.y == key && j + 1 < i) + (k.z == key && j + 2 < i) + (k.w == key && j + 3 < i);
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

// More: by digits from the lowest, two launches for each. (Counting the next digit at the tokens' new places in the launch that moves
// them, by atomics, took 10 us more of it, and the launch that it saves takes 5.)
struct SortArgs {
  const int* tokens;
  const unsigned* keys;  // sorted by lower digits, with their places; the first pass reads the tokens themselves
  const int* places;
  unsigned* keys_out;
  int* places_out;
  int* counts;  // [blocks][2^bits]
  int* marks;   // see FillArgs; or NULL
  int count, vocab, blocks, each, shift, bits;  // each: tokens of a block, a multiple of ST
};

template <bool FIRST>
__global__ __launch_bounds__(ST) void sort_count_kernel(SortArgs a, FillArgs fill) {
  if (fills(fill)) return;
  __shared__ int n[1 << kDigit];
  const int digits = 1 << a.bits, tid = threadIdx.x, b = blockIdx.x;
  for (int d = tid; d < digits; d += ST) n[d] = 0;
  __syncthreads();
  for (int r = 0; r < a.each; r += ST) {
    const long long i = (long long)b * a.each + r + tid;
    if (i < a.count) {
      const unsigned key = FIRST ? key_of(a.tokens[i], a.vocab) : a.keys[i];
      atomicAdd(&n[key >> a.shift & (digits - 1)], 1);
      if (FIRST && a.marks && key < (unsigned)a.vocab) a.marks[key] = (int)i;
    }
  }
  __syncthreads();
  for (int d = tid; d < digits; d += ST) a.counts[b * digits + d] = n[d];
}

template <bool FIRST>
__global__ __launch_bounds__(ST) void sort_move_kernel(SortArgs a, FillArgs fill) {
  if (fills(fill)) return;
  constexpr int WAVES = ST / 64;
  __shared__ int to[WAVES][1 << kDigit];  // where a wave's next token of a digit goes
  __shared__ int sums[WAVES];
  const int digits = 1 << a.bits, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, b = blockIdx.x;
  const auto key_at = [&](long long i) { return FIRST ? key_of(a.tokens[i], a.vocab) : a.keys[i]; };
  // A digit's tokens in the blocks before this one, and in all, by as many groups of threads as there are for each digit.
  int before = 0, all = 0;
  for (int k = tid >> a.bits; k < a.blocks; k += (ST >> a.bits) * 8) {
    int n[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const int at = k + u * (ST >> a.bits);
      n[u] = at < a.blocks ? a.counts[at * digits + (tid & (digits - 1))] : 0;
    }
#pragma unroll
    for (int u = 0; u < 8; u++) {
      before += k + u * (ST >> a.bits) < b ? n[u] : 0;
      all += n[u];
    }
  }
  int* room = &to[0][0];  // (two numbers a thread)
  room[tid] = before;
  room[ST + tid] = all;
  __syncthreads();
  before = all = 0;
  if (tid < digits)
    for (int k = tid; k < ST; k += digits) {
      before += room[k];
      all += room[ST + k];
    }
  __syncthreads();
  for (int d = tid; d < digits * WAVES; d += ST) to[d >> a.bits][d & (digits - 1)] = 0;
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
  int count, vocab, channels, ranges, each, slabs, sum_groups, accumulate, filled;  // slabs: of a row's columns; sum_groups: workgroups that sum
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

// A lane's vector, whose elements below `least` are the one's before too.
template <typename G, int V>
__device__ __forceinline__ void put_vector(G* p, int least, const float (&sum)[V], float scale, int accumulate) {
  if (V > 1 && least > 0 && accumulate) {  // (what is shared is added to once)
#pragma unroll
    for (int j = 0; j < V; j++)
      if (j >= least) p[j] = to_t<G>(__builtin_fmaf(sum[j], scale, (float)p[j]));
  } else {
    put<G, V>(p, V, sum, scale, accumulate);
  }
}

// The first sorted place whose key is at least `key`, by seven probes at a time: each step waits for memory.
__device__ __forceinline__ int lower_bound(const unsigned* keys, int count, unsigned key) {
  int lo = 0, hi = count;
  while (lo < hi) {
    const int step = (hi - lo + 7) / 8;
    int below = 0;
#pragma unroll
    for (int t = 1; t < 8; t++) {
      const int at = lo + t * step - 1;
      below += at < hi && keys[min(at, hi - 1)] < key;
    }
    lo += below * step;
    if (below < 7) hi = min(hi, lo + step - 1);
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

typedef unsigned short u16x4_any __attribute__((ext_vector_type(4), aligned(2)));
// V elements of a row, as they were read.
template <typename T, int V>
struct Columns {
  typename RowVec<T>::type raw;
  __device__ __forceinline__ void load(const T* p) { raw = *(const typename RowVec<T>::type*)p; }
  __device__ __forceinline__ float at(int j) const { return widen1<T>(raw, j); }
};
template <>
struct Columns<f16, 4> {
  u16x4_any raw;
  __device__ __forceinline__ void load(const f16* p) { raw = *(const u16x4_any*)p; }
  __device__ __forceinline__ float at(int j) const { return (float)__builtin_bit_cast(f16, (unsigned short)raw[j]); }
};
template <>
struct Columns<bf16, 4> {
  u16x4_any raw;
  __device__ __forceinline__ void load(const bf16* p) { raw = *(const u16x4_any*)p; }
  __device__ __forceinline__ float at(int j) const { return __uint_as_float((unsigned)raw[j] << 16); }
};
template <typename T>
struct Columns<T, 1> {
  T raw;
  __device__ __forceinline__ void load(const T* p) { raw = *p; }
  __device__ __forceinline__ float at(int) const { return (float)raw; }
};

// A workgroup for L vectors of V elements over a range: L lanes take a share of its tokens each. A run that
// reaches over the ends of a share is added up in LDS; only one that reaches over the range's ends is left to the second launch. The
// workgroups behind fill.
template <typename T, typename G, int V, int L>
__global__ __launch_bounds__(ET) void embedding_sums_kernel(SumArgs a) {
  constexpr int AT_ONCE = 4, SHARES = ET / L;
  if ((int)blockIdx.x >= a.sum_groups) {
    fill_rows<G>(a, __builtin_amdgcn_readfirstlane((blockIdx.x - a.sum_groups) * (ET / 64) + (threadIdx.x >> 6)),
                 (gridDim.x - a.sum_groups) * (ET / 64));
    return;
  }
  __shared__ float ends[V][ET];     // a share's sum of a run from before it
  __shared__ int firsts[SHARES];    // the first key of each share, -1 where it has no token
  const int tid = threadIdx.x, share = L == 64 ? __builtin_amdgcn_readfirstlane(tid / L) : tid / L;
  const int range = blockIdx.x / a.slabs, column = ((blockIdx.x - range * a.slabs) * L + tid % L) * V;
  const bool in = column < a.channels;
  const int c = min(column, a.channels - V), least = column - c;  // elements below `least` are the vector's before
  const int begin = range * a.each, end = min(begin + a.each, a.count), each = a.each / SHARES;
  const int first = begin + share * each, last = min(first + each, end);
  const T* dy = (const T*)a.dy + c;
  float sum[V] = {};
  int run = -1;
  bool before = false;
  const auto write = [&](int key) {
    if (in) put_vector<G, V>((G*)a.grad + (size_t)key * a.ld_grad + c, least, sum, a.scale, a.accumulate);
  };
  const auto keep = [&] {
#pragma unroll
    for (int j = 0; j < V; j++) ends[j][tid] = sum[j];
  };
  bool tail = false;  // a run that begins in this share goes on behind it
  if (first < last) {
    run = (int)a.keys[first];
    before = first > 0 && (int)a.keys[first - 1] == run;
    const int next = last < a.count ? (int)a.keys[last] : -1;
    if (tid % L == 0) firsts[share] = run;
    // Four tokens' columns are under way while those of the four before are added, and the keys and places of the four behind: a wait for
    // what was asked for earlier does not wait for the sums written since. (Every lane of a share reads the same four; a share begins at a
    // multiple of four. Keys past the last lie within the workspace.)
    int4 key[2], place, keys_ahead, places_ahead;
    Columns<T, V> f[2][AT_ONCE];
    const auto look = [&](int i0) {
      if (i0 >= last) return;
      keys_ahead = *(const int4*)(a.keys + i0);
      places_ahead = *(const int4*)(a.places + i0);
    };
    const auto ask = [&](int i0, int4& k, Columns<T, V>(&to)[AT_ONCE]) {
      k = int4{a.vocab, a.vocab, a.vocab, a.vocab};
      if (i0 >= last) return;
      k = keys_ahead;
      place = places_ahead;
      if (i0 + 1 >= last) k.y = a.vocab;
      if (i0 + 2 >= last) k.z = a.vocab;
      if (i0 + 3 >= last) k.w = a.vocab;
      if (!in) return;
      if (k.x < a.vocab) to[0].load(dy + (size_t)place.x * a.ld);
      if (k.y < a.vocab) to[1].load(dy + (size_t)place.y * a.ld);
      if (k.z < a.vocab) to[2].load(dy + (size_t)place.z * a.ld);
      if (k.w < a.vocab) to[3].load(dy + (size_t)place.w * a.ld);
    };
    const auto add = [&](int k, const Columns<T, V>& from) {
      if (k >= a.vocab) return;
      if (k != run) {
        if (before) keep();
        else write(run);
#pragma unroll
        for (int j = 0; j < V; j++) sum[j] = 0.f;
        run = k;
        before = false;
      }
#pragma unroll
      for (int j = 0; j < V; j++) sum[j] += from.at(j);
    };
    look(first);
    ask(first, key[0], f[0]);
    look(first + AT_ONCE);
    for (int i0 = first; i0 < last; i0 += 2 * AT_ONCE) {
#pragma unroll
      for (int side = 0; side < 2; side++) {
        const int i = i0 + side * AT_ONCE;
        ask(i + AT_ONCE, key[1 - side], f[1 - side]);
        look(i + 2 * AT_ONCE);
        add(key[side].x, f[side][0]);
        add(key[side].y, f[side][1]);
        add(key[side].z, f[side][2]);
        add(key[side].w, f[side][3]);
      }
    }
    if (run < a.vocab) {
      tail = !before && next == run;
      if (before) keep();
      else if (!tail) write(run);
    }
  } else if (tid % L == 0) {
    firsts[share] = -1;
  }
  __syncthreads();
  // The first share's run from before the range, and each share's run that goes on: with its parts in the shares behind.
  const bool from_before = share == 0 && first < last && first > 0 && firsts[0] < a.vocab && (int)a.keys[first - 1] == firsts[0];
  const auto collect = [&](int key) {
    int s = share + 1;
    for (; s < SHARES && firsts[s] == key; s++) {
#pragma unroll
      for (int j = 0; j < V; j++) sum[j] += ends[j][s * L + tid % L];
    }
    return (s == SHARES || begin + s * each >= end) && end < a.count && (int)a.keys[end] == key;  // goes on behind the range
  };
  const auto leave = [&](int side) {
    if (in) put<float, V>(a.parts + ((size_t)range * 2 + side) * a.channels + c, V, sum, 1.f, 0);
  };
  if (tail) {
    if (collect(run)) leave(1);
    else write(run);
  }
  if (from_before) {
    const int key = firsts[0];
#pragma unroll
    for (int j = 0; j < V; j++) sum[j] = ends[j][tid];
    collect(key);  // (with the shares behind that begin with it)
    leave(0);
  }
}

// Runs over several ranges: a workgroup for up to JS slabs of 256 channels of each range that such a run begins in. Its waves are
// `wide` slabs side by side, and share the ranges where there are fewer.
constexpr int JT = 512, JS = JT / 64;
template <typename G>
__global__ __launch_bounds__(JT) void embedding_join_kernel(SumArgs a, int blocks, int wide) {
  __shared__ float4 joined[JS][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slab = w & (wide - 1), step = JS / wide;
  const long long all = (long long)(a.ranges - 1) * blocks;
  for (long long id = blockIdx.x; id < all; id += gridDim.x) {
    const int range = (int)(id / blocks), c = ((int)(id - (long long)range * blocks) * JS + slab) * 256 + lane * 4;
    const int first = range * a.each, last = first + a.each;  // (one more range follows)
    const unsigned key = a.keys[last], at_first = a.keys[first], at_last = a.keys[last - 1], ahead = first > 0 ? a.keys[first - 1] : ~0u;
    if (key >= (unsigned)a.vocab || at_last != key) continue;
    if (at_first == key && ahead == key) continue;  // begins before
    int ends = range + 1;  // the last range with its tokens: 64 ranges' first keys at a time
    for (int r = range + 2; r < a.ranges; r += 64) {
      const unsigned long long others = __ballot(r + lane >= a.ranges || a.keys[min(r + lane, a.ranges - 1) * a.each] != key);
      ends = r + (others ? __ffsll(others) - 1 : 64) - 1;
      if (others) break;
    }
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    const int left = max(a.channels - c, 0);
#pragma unroll 4
    for (int r = range + w / wide; r <= ends; r += step) {
      float f[4];
      load_vec<float>(a.parts + ((size_t)r * 2 + (r == range)) * a.channels + c, left, f);
#pragma unroll
      for (int j = 0; j < 4; j++) sum[j] += (double)f[j];
    }
    // (A share's sum is rounded to float here; at most JS of them make the row's.)
    joined[w][lane] = float4{(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]};
    __syncthreads();
    if (w < wide) {
      for (int j = 0; j < 4; j++) sum[j] = 0.0;
      for (int k = w; k < JS; k += wide) {
        const float4 f = joined[k][lane];
        sum[0] += f.x;
        sum[1] += f.y;
        sum[2] += f.z;
        sum[3] += f.w;
      }
      const float f[4] = {(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]};
      put<G, 4>((G*)a.grad + (size_t)key * a.ld_grad + c, left, f, a.scale, a.accumulate);
    }
    __syncthreads();
  }
}

// Few tokens of a small table, in one launch: a workgroup for a slab of a few rows of the table finds their tokens by itself. It counts and
// places them as the sort does, rows for digits; then L lanes take a row of few tokens each, and all of them one of many. 722 tokens of
// 362 rows of 384 floats take 4 us of a graph (10 where they are all the same), 11 by the launches below; but of larger tables, where a
// workgroup has more rows than it takes at once, 1024 skewed tokens of 16384 rows of 512 bf16 16 and 14.
constexpr int NT = 1024, kFewTokens = NT, kFewRows = 16, kFewOfRow = 16;
struct FewArgs {
  const int* tokens;
  const void* dy;
  void* grad;
  long long ld, ld_grad;
  int count, vocab, channels, rows, slabs, lanes, accumulate;  // rows: of a workgroup; lanes: 2^lanes = L
  float scale;
};
template <typename T, typename G, int V>
__global__ __launch_bounds__(NT) void embedding_few_kernel(FewArgs a) {
  constexpr int WAVES = NT / 64, AT_ONCE = 8;
  __shared__ int to[WAVES][kFewRows];  // where a wave's tokens of a row go
  __shared__ int firsts[kFewRows + 1], places[kFewTokens];
  __shared__ float joined[V][NT];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int range = blockIdx.x / a.slabs, row0 = range * a.rows, rows = min(a.rows, a.vocab - row0);
  // (A token before row0, or outside the table, is past `rows` as an unsigned difference.)
  const unsigned row = tid < a.count ? (unsigned)a.tokens[tid] - (unsigned)row0 : ~0u;
  const bool mine = row < (unsigned)rows;
  if (lane < kFewRows) to[w][lane] = 0;
  __syncthreads();
  if (mine) atomicAdd(&to[w][row], 1);
  __syncthreads();
  if (tid < kFewRows) {
    int n = 0;
    for (int k = 0; k < WAVES; k++) {
      const int here = to[k][tid];
      to[k][tid] = n;
      n += here;
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < kFewRows; o <<= 1) {
      const int v = __shfl_up(upto, o);
      upto += lane >= o ? v : 0;
    }
    firsts[tid + 1] = upto;
    if (tid == 0) firsts[0] = 0;
    for (int k = 0; k < WAVES; k++) to[k][tid] += upto - n;
  }
  __syncthreads();
  unsigned long long same = __ballot(mine);
  for (int k = 0; 1 << k < kFewRows; k++) {
    const unsigned long long set = __ballot(row >> k & 1);
    same &= row >> k & 1 ? set : ~set;
  }
  if (mine) places[to[w][row] + __popcll(same & ((1ull << lane) - 1))] = tid;
  __syncthreads();

  const int L = 1 << a.lanes, share = tid >> a.lanes, shares = NT >> a.lanes;
  const int column = ((blockIdx.x - range * a.slabs) * L + (tid & (L - 1))) * V;
  const bool in = column < a.channels;
  const int c = min(column, a.channels - V), least = column - c;  // elements below `least` are the vector's before
  const T* dy = (const T*)a.dy + c;
  const auto add_up = [&](int first, int last, float(&sum)[V]) {
#pragma unroll
    for (int j = 0; j < V; j++) sum[j] = 0.f;
    for (int i = first; i < last; i += AT_ONCE) {
      Columns<T, V> f[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; k++)
        if (i + k < last) f[k].load(dy + (size_t)places[i + k] * a.ld);
#pragma unroll
      for (int k = 0; k < AT_ONCE; k++) {
        if (i + k >= last) break;
#pragma unroll
        for (int j = 0; j < V; j++) sum[j] += f[k].at(j);
      }
    }
  };
  const auto write = [&](int r, const float(&sum)[V]) {
    if (in) put_vector<G, V>((G*)a.grad + (size_t)(row0 + r) * a.ld_grad + c, least, sum, a.scale, a.accumulate);
  };
  for (int r = share; r < rows; r += shares) {
    const int first = firsts[r], last = firsts[r + 1];
    if (last - first > kFewOfRow || (a.accumulate && first == last)) continue;
    float sum[V];
    add_up(first, last, sum);
    write(r, sum);
  }
  for (int r = 0; r < rows; r++) {
    const int first = firsts[r], n = firsts[r + 1] - first;
    if (n <= kFewOfRow) continue;
    const int each = (n + shares - 1) / shares, used = (n + each - 1) / each, begin = first + share * each;
    float sum[V];
    add_up(begin, min(begin + each, first + n), sum);
#pragma unroll
    for (int j = 0; j < V; j++) joined[j][tid] = sum[j];
    __syncthreads();
    if (share == 0) {
#pragma unroll 4
      for (int k = 1; k < used; k++) {
#pragma unroll
        for (int j = 0; j < V; j++) sum[j] += joined[j][(k << a.lanes) + tid];
      }
      write(r, sum);
    }
    __syncthreads();
  }
}

// How the tokens are sorted and cut, and where their parts of the workspace lie.
struct Plan {
  int passes, bits, blocks, each_block, each, ranges;  // passes: 0 where the tokens are ranked
  bool marked;  // rows that no token names are filled by marks
  size_t keys, places, counts, marks, parts, bytes;
};
// From one copy of the keys to the other: whole eights, which are read at once.
size_t plan_stride(int count) { return ((size_t)count + 7) / 8 * 8; }
// Lanes for a slab of `chunks` vectors.
int lanes_of(int chunks) {
  int lanes = 1;
  while (lanes < chunks && lanes < 64) lanes *= 2;
  return lanes;
}
// (A range is ET / lanes shares of tokens that leave some 4096 waves, 8 tokens at least and 64 at most, a multiple of 8, for the type whose
// rows take the fewest lanes: ranges, and with them the workspace, are the same for every type. Where the sums' launch has other lanes a row, its
// shares are as many times longer or shorter: 4 to 256 tokens, a multiple of 4.)
Plan plan_of(int count, int vocab, int channels) {
  Plan p = {};
  if (count > kRanked) {
    const int bits = 32 - __builtin_clz((unsigned)vocab);  // of the keys 0 ... vocab
    p.passes = (bits + kDigit - 1) / kDigit;
    // (Six at least: a launch adds a digit's counts up by as many threads as there are digits, 11552 tokens of 3 rows 16 us with 2 bits.)
    p.bits = std::max((bits + p.passes - 1) / p.passes, 6);
    const long long rounds = ((long long)count + (long long)ST * kMostBlocks - 1) / ((long long)ST * kMostBlocks);
    p.each_block = (int)(rounds * ST);
    p.blocks = (int)(((long long)count + p.each_block - 1) / p.each_block);
  }
  const int chunks = channels < 4 ? 8 : (channels + 7) / 8, lanes = channels < 4 ? 8 : channels < 8 ? 2 : lanes_of(chunks);
  const long long waves = (long long)count * ((chunks + lanes - 1) / lanes) * lanes / 64;  // one token each
  p.each = (int)std::min(std::max(waves / 4096 / 8 * 8, 8ll), 64ll) * (ET / lanes);
  p.ranges = (int)(((long long)count + p.each - 1) / p.each);
  const auto room = [&](size_t n) {
    const size_t at = p.bytes;
    p.bytes += (n + 255) / 256 * 256;
    return at;
  };
  const size_t copies = p.passes > 1 ? 2 : 1;
  p.keys = room(copies * plan_stride(count) * 4);
  p.places = room(copies * plan_stride(count) * 4);
  p.counts = room((size_t)p.blocks * (4 << p.bits));
  // (Fewer: see FillArgs. More leave few rows without a token, and write each mark over and over: 1000000 tokens of 5000 rows 96 us, 92.)
  p.marked = p.passes && count > vocab / 4 && count / 4 <= vocab;
  p.marks = room(p.marked ? (size_t)vocab * 4 : 0);
  p.parts = room((size_t)p.ranges * 2 * channels * 4);
  return p;
}

inline int grid_of(long long threads) { return (int)std::min((threads + ET - 1) / ET, 1ll << 20); }

// filled: whether the launches fill rows.
void sort_tokens(const kg_embedding_args& a, const Plan& plan, SumArgs& p, bool filled, hipStream_t s) {
  char* w = (char*)a.workspace;
  unsigned* keys = (unsigned*)(w + plan.keys);
  int* places = (int*)(w + plan.places);
  p.keys = keys;
  p.places = places;
  FillArgs fill = {};
  fill.groups = plan.passes ? plan.blocks : (a.count + RI - 1) / RI;
  const int size = a.grad_type == PREC_F32 ? 4 : 2, launches = plan.passes ? 2 * plan.passes : 1;
  fill.grad = a.grad; fill.ld = a.ld_grad * size; fill.bytes = (long long)a.channels * size;
  // The grid of the next launch, with its share of the rows: none for the one that leaves the marks.
  const bool marks = filled && plan.marked;
  if (marks) {
    fill.marks = (const int*)(w + plan.marks);
    fill.tokens = a.tokens;
    fill.count = a.count;
  }
  const auto grid = [&](int launch) {
    const auto upto = [&](int k) { return k < marks ? 0 : (int)((long long)a.vocab * (k - marks) / (launches - marks)); };
    fill.first = upto(launch);
    fill.rows = filled ? upto(launch + 1) - fill.first : 0;
    const int each = marks ? kMarked * (ST / 64) : ST / 64;
    return dim3(fill.groups + std::min((fill.rows + each - 1) / each, 512));
  };
  if (!plan.passes) {
    const dim3 all = grid(0);
    launch_k(sort_rank_kernel, all, ST, 0, s, a.tokens, keys, places, a.count, a.vocab, fill);
    return;
  }
  SortArgs t = {};
  t.tokens = a.tokens;
  t.counts = (int*)(w + plan.counts);
  t.marks = marks ? (int*)(w + plan.marks) : nullptr;
  t.count = a.count; t.vocab = a.vocab; t.blocks = plan.blocks; t.each = plan.each_block; t.bits = plan.bits;
  for (int k = 0; k < plan.passes; k++) {
    t.shift = k * plan.bits;
    t.keys_out = keys + (size_t)(k & 1) * plan_stride(a.count);
    t.places_out = places + (size_t)(k & 1) * plan_stride(a.count);
    dim3 all = grid(2 * k);
    if (k == 0) launch_k(sort_count_kernel<true>, all, ST, 0, s, t, fill);
    else launch_k(sort_count_kernel<false>, all, ST, 0, s, t, fill);
    all = grid(2 * k + 1);
    if (k == 0) launch_k(sort_move_kernel<true>, all, ST, 0, s, t, fill);
    else launch_k(sort_move_kernel<false>, all, ST, 0, s, t, fill);
    p.keys = t.keys = t.keys_out;
    p.places = t.places = t.places_out;
  }
}

template <typename T, typename G, int V, int L>
void sums(SumArgs p, int chunks, hipStream_t s) {
  p.slabs = (chunks + L - 1) / L;
  p.sum_groups = p.ranges * p.slabs;
  const int fill = p.accumulate || p.filled ? 0 : (int)std::min(((long long)p.vocab + FR * ET / 64 - 1) / (FR * ET / 64), 8192ll);
  if (p.sum_groups + fill) launch_k(embedding_sums_kernel<T, G, V, L>, dim3(p.sum_groups + fill), ET, 0, s, p);
  if (p.ranges > 1) {
    const int blocks = (int)(((long long)p.channels + 256 * JS - 1) / (256 * JS));
    const int wide = p.channels <= 256 ? 1 : p.channels <= 512 ? 2 : p.channels <= 1024 ? 4 : JS;
    launch_k(embedding_join_kernel<G>, dim3((int)std::min((long long)(p.ranges - 1) * blocks, 1ll << 20)), JT, 0, s, p, blocks, wide);
  }
}
template <typename T, typename G>
void backward_typed(const SumArgs& p, hipStream_t s) {
  // (As many elements a lane as it stores in 16 bytes: with eight, a wave's stores of floats were halves of what it has, 65536 tokens of
  // 1024 bf16 channels into floats 64 us of the sums' launch, now 57.)
  constexpr int V = kVec<G>;
  if (p.channels < V) return sums<T, G, 1, 8>(p, p.channels, s);
  const int chunks = (int)(((long long)p.channels + V - 1) / V);
  switch (lanes_of(chunks)) {
    case 1: return sums<T, G, V, 1>(p, chunks, s);
    case 2: return sums<T, G, V, 2>(p, chunks, s);
    case 4: return sums<T, G, V, 4>(p, chunks, s);
    case 8: return sums<T, G, V, 8>(p, chunks, s);
    case 16: return sums<T, G, V, 16>(p, chunks, s);
    case 32: return sums<T, G, V, 32>(p, chunks, s);
    default: return sums<T, G, V, 64>(p, chunks, s);
  }
}

// Returns whether there are few tokens, and the launch.
template <typename T, typename G>
bool few(const SumArgs& p, const int* tokens, hipStream_t s) {
  constexpr int V = kVec<G>;
  const bool narrow = p.channels < V;
  FewArgs a = {};
  a.lanes = 3;
  const long long chunks = narrow ? p.channels : ((long long)p.channels + V - 1) / V;
  while (1 << a.lanes < chunks && a.lanes < 6) a.lanes++;
  const long long slabs = (chunks + (1 << a.lanes) - 1) >> a.lanes, groups = slabs * p.vocab;  // a row each
  if (p.count > kFewTokens || groups > 512 * kFewRows) return false;
  a.tokens = tokens;
  a.dy = p.dy; a.ld = p.ld;
  a.grad = p.grad; a.ld_grad = p.ld_grad;
  a.count = p.count; a.vocab = p.vocab; a.channels = p.channels; a.accumulate = p.accumulate; a.scale = p.scale;
  a.rows = (int)((groups + 511) / 512);
  a.slabs = (int)slabs;
  const dim3 grid((p.vocab + a.rows - 1) / a.rows * a.slabs);
  if (narrow) launch_k(embedding_few_kernel<T, G, 1>, grid, NT, 0, s, a);
  else launch_k(embedding_few_kernel<T, G, V>, grid, NT, 0, s, a);
  return true;
}

}  // namespace

size_t embedding_backward_workspace(int count, int vocab, int channels) { return count < 1 ? 0 : plan_of(count, vocab, channels).bytes; }

void launch_embedding(const kg_embedding_args& a, hipStream_t s) {
  const float scale = (float)a.scale;
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    constexpr int V = kVec<T>;
    const auto run = [&](auto kernel, int vec, int each) {
      const int chunks = (a.channels + vec - 1) / vec;
      const long long threads = ((long long)a.count + each - 1) / each * chunks;
      const int past = (long long)a.count * a.channels * (long long)sizeof(T) > kPastBytes;
      launch_k(kernel, dim3(grid_of(threads)), ET, 0, s, a.tokens, (const T*)a.table, (T*)a.y, a.ld_table, a.ld_y, a.count, a.vocab,
               a.channels, chunks, scale, past);
    };
    const bool few = (long long)a.count * ((a.channels + V - 1) / V) < kFewColumns;
    if (a.channels < V) run(embedding_kernel<T, 1, 4>, 1, 4);
    else if (few) run(embedding_kernel<T, V, 1>, V, 1);
    else run(embedding_kernel<T, V, 4>, V, 4);
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
  const auto go = [&](auto of_dy, auto of_grad) {
    using T = decltype(of_dy);
    using G = decltype(of_grad);
    if (few<T, G>(p, a.tokens, s)) return;
    if (a.count) {
      const Plan plan = plan_of(a.count, a.vocab, a.channels);
      p.parts = (float*)((char*)a.workspace + plan.parts);
      p.ranges = plan.ranges;
      p.each = plan.each;
      // (A table of up to 64 MB is filled within the sort's time.)
      const long long bytes = (long long)a.vocab * a.channels * (long long)sizeof(G);
      p.filled = !p.accumulate && (plan.marked || bytes <= 64ll << 20 || a.count <= a.vocab / 4);
      sort_tokens(a, plan, p, p.filled, s);
    }
    backward_typed<T, G>(p, s);
  };
  if (a.type == PREC_F32) go(0.f, 0.f);
  else if (a.type == PREC_F16 && a.grad_type == a.type) go((f16)0.f, (f16)0.f);
  else if (a.type == PREC_F16) go((f16)0.f, 0.f);
  else if (a.grad_type == a.type) go((bf16)0.f, (bf16)0.f);
  else go((bf16)0.f, 0.f);
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
