// The AdamW step over many tensors at once (kg_adamw_step), with moments in 32 or in 8 bits, and the moments as numbers.
//
// Bound by memory: 28 bytes an element in float, 16 with 16-bit parameters and gradients, float masters and 8-bit moments. A step
// of 29 M float elements in 310 tensors takes 144 us (5.6 TB/s), one of 240 M bf16 with masters and 8 bits 710 (5.4 TB/s).
// One launch covers up to kTensors tensors, whose descriptions travel as kernel arguments: nothing has to be uploaded, and a
// captured launch carries them. Each workgroup takes kChunk consecutive elements of one tensor.
//
// 8 bits: a block of 256 elements is one wave, four elements a lane, so that its largest moment is a wave's reduction. A
// block's unit is a power of two: scaling by it is exact, and so is every step of the rounding (the quotient by a code's
// spacing, its floor, the comparison with the random part), which makes the codes a function of the moments alone. The file
// is compiled without contraction into fused multiply-adds, so that the moments before the rounding are each formula's
// plain sequence of float operations.
#include "kgx_device.h"
#include <climits>

#include "kgx_learn.h"

namespace kgx {

namespace {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32_any __attribute__((aligned(1)));

constexpr int kTensors = 111;                // descriptions in the 4 KB of kernel arguments
constexpr int kBlock = KG_ADAMW_BLOCK;
constexpr int kUnroll = 4, kWaves = 4;       // blocks a wave, waves a workgroup
constexpr int kChunk = kBlock * kUnroll * kWaves;

struct AdamTensor {
  void* param;
  const void* grad;
  float* master;
  long long elements, first_block;
  float weight_decay;
  short param_type, grad_type;
};
// The same in 32 bytes: addresses have 48 bits, a piece up to 2^34 elements, a state up to 2^39 blocks. (400 small tensors then
// take four launches, which wait for each other, for six of 72 descriptions of 48 bytes: 18.5 us for 24.4; 310 tensors of 29 M
// floats 145 for 152.)
struct AdamPacked {
  unsigned long long word[4];
  static AdamPacked of(const AdamTensor& t) {
    const unsigned long long n = (unsigned long long)t.elements, b = (unsigned long long)t.first_block;
    return {{(unsigned long long)t.param | n << 48, (unsigned long long)t.grad | (n >> 16) << 48,
             (unsigned long long)t.master | (n >> 32 | (unsigned long long)t.param_type << 3 | (unsigned long long)t.grad_type << 5 | (b >> 32) << 7) << 48,
             (b & 0xffffffffu) | (unsigned long long)__builtin_bit_cast(unsigned, t.weight_decay) << 32}};
  }
  __device__ __forceinline__ AdamTensor open() const {
    constexpr unsigned long long address = (1ull << 48) - 1;
    const unsigned top = (unsigned)(word[2] >> 48);
    AdamTensor t;
    t.param = (void*)(word[0] & address);
    t.grad = (const void*)(word[1] & address);
    t.master = (float*)(word[2] & address);
    t.elements = (long long)(word[0] >> 48 | (word[1] >> 48) << 16 | (unsigned long long)(top & 7) << 32);
    t.first_block = (long long)((word[3] & 0xffffffffu) | (unsigned long long)(top >> 7) << 32);
    t.weight_decay = __uint_as_float((unsigned)(word[3] >> 32));
    t.param_type = (short)(top >> 3 & 3);
    t.grad_type = (short)(top >> 5 & 3);
    return t;
  }
};
static_assert(PREC_F32 >= 0 && PREC_F32 < 4 && PREC_F16 >= 0 && PREC_F16 < 4 && PREC_BF16 >= 0 && PREC_BF16 < 4, "two bits a type");
struct AdamArgs {
  AdamPacked t[kTensors];
  int start[kTensors];  // first workgroup of tensor i; INT_MAX past the last
  kg_adamw_values_t values;
  const kg_adamw_values_t* device_values;
  void *m, *v;
  unsigned char *m_exp, *v_exp;
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

// Four elements at index i of a tensor of any element type. WHOLE: they are all there; else elements from n on read as 0 and
// are not written. (Past the caches: every byte of a step is touched once, and with 29M float elements that took 157 us
// where plain accesses took 180.)
template <bool WHOLE>
__device__ __forceinline__ floatx4 load4(const void* p, int type, long long i, long long n) {
  floatx4 f = {0.f, 0.f, 0.f, 0.f};
  if (WHOLE || i + 4 <= n) {
    if (type == PREC_F32) {
      f = __builtin_nontemporal_load((const f32x4_any*)((const float*)p + i));
    } else {
      const u16x4_any h = __builtin_nontemporal_load((const u16x4_any*)((const unsigned short*)p + i));
#pragma unroll
      for (int j = 0; j < 4; j++)
        f[j] = type == PREC_BF16 ? __uint_as_float((unsigned)h[j] << 16) : (float)__builtin_bit_cast(f16, (unsigned short)h[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j < n)
        f[j] = type == PREC_F32 ? ((const float*)p)[i + j]
                                : type == PREC_BF16 ? (float)((const bf16*)p)[i + j] : (float)((const f16*)p)[i + j];
  }
  return f;
}
template <bool WHOLE>
__device__ __forceinline__ void store4_any(void* p, int type, long long i, long long n, floatx4 f) {
  if (WHOLE || i + 4 <= n) {
    if (type == PREC_F32) {
      __builtin_nontemporal_store((f32x4_any)f, (f32x4_any*)((float*)p + i));
    } else {
      u16x4_any h;
#pragma unroll
      for (int j = 0; j < 4; j++)
        h[j] = type == PREC_BF16 ? __builtin_bit_cast(unsigned short, (bf16)f[j]) : __builtin_bit_cast(unsigned short, (f16)f[j]);
      __builtin_nontemporal_store(h, (u16x4_any*)((unsigned short*)p + i));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j < n) {
        if (type == PREC_F32) ((float*)p)[i + j] = f[j];
        else if (type == PREC_BF16) ((bf16*)p)[i + j] = (bf16)f[j];
        else ((f16*)p)[i + j] = (f16)f[j];
      }
  }
}

// A 32-bit hash: two rounds of a shift and an odd multiplier (the fraction of the golden ratio and of e). 16 bits each round
// the first and the second moment.
__device__ __forceinline__ unsigned mix32(unsigned x) {
  x = (x ^ (x >> 16)) * 0x9E3779B9u;
  x = (x ^ (x >> 15)) * 0xB7E15163u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ float exp_bits(int e) { return __uint_as_float((unsigned)e << 23); }
// The unit of a block: 2^(exp - bias), NaN where the block held something that was no number. (A new state's exponents
// are 0, below the least that a step writes.)
__device__ __forceinline__ float unit_of(int exp, int bias) {
  const int e = exp - bias + 127;
  return exp == 255 ? __uint_as_float(0x7fc00000u) : exp_bits(e < 1 ? 1 : e);
}
// The exponent of a block whose largest magnitude has the bits `top`: the least unit in which it does not pass the largest
// code (mantissas above it, `carry` short of the next power of two, go there).
__device__ __forceinline__ int exp_of(unsigned top, unsigned carry, int least) {
  const int e = (int)((top + carry) >> 23);
  return e < least ? least : e > 255 ? 255 : e;
}

// The correctly rounded root: the hardware's (an ulp), or the neighbour below or above it by the sign of what their product with
// it leaves of v. 0, infinity and NaN keep the hardware's: every comparison fails. Below 2^-96 what they leave underflows, and the
// hardware takes subnormal numbers for 0: those are scaled by 2^64 first, their roots by 2^-32. (Few steps have one, so the four of
// a lane are tested together, for scaling each argument would be seven of nineteen operations.)
__device__ __forceinline__ float root_of(float v) {
  const float s = __builtin_amdgcn_sqrtf(v);
  const float below = __uint_as_float(__float_as_uint(s) - 1), above = __uint_as_float(__float_as_uint(s) + 1);
  float r = __builtin_fmaf(-below, s, v) <= 0.f ? below : s;
  return __builtin_fmaf(-above, s, v) > 0.f ? above : r;
}
__device__ __forceinline__ floatx4 roots_of(const floatx4& v) {
  floatx4 r;
  unsigned least = ~0u;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    r[j] = root_of(v[j]);
    least = min(least, __float_as_uint(v[j]) - 1);  // (0 needs no scaling)
  }
  if (least < __float_as_uint(0x1p-96f) - 1) {
#pragma unroll
    for (int j = 0; j < 4; j++) r[j] = v[j] < 0x1p-96f ? root_of(v[j] * 0x1p64f) * 0x1p-32f : r[j];
  }
  return r;
}

constexpr int M_BIAS = 135, M_LEAST = 9, V_BIAS = 138, V_LEAST = 12;
constexpr unsigned M_CARRY = 0x1FFFFF, V_CARRY = 0x03FFFF;  // largest codes 1.75 and 1.96875 times a power of two

// A code is the quotient of its value y, in the block's units, by the spacing there, rounded up where the cut part exceeds
// u / 2^16, u its random part. In the codes' normal range the quotient is the top of y's mantissa and the code the top of its
// bits, less the bias: one addition rounds. Below it the spacing is that of the least codes.
// e4m3 without its sign; normal from 2^-6 on.
__device__ __forceinline__ unsigned encode_m_normal(float y, unsigned u) { return ((__float_as_uint(y) + (u << 4)) >> 20) - (120u << 3); }
__device__ __forceinline__ unsigned encode_m_low(float y, unsigned u) { return (unsigned)(y * 512.f + (float)u * 0x1p-16f); }
// e3m5; normal from 32 on. A positive value never becomes 0.
__device__ __forceinline__ unsigned encode_v_normal(float y, unsigned u) { return ((__float_as_uint(y) + (u << 2)) >> 18) - (131u << 5); }
__device__ __forceinline__ unsigned encode_v_low(float y, unsigned u) {
  const unsigned n = (unsigned)(y + (float)u * 0x1p-16f);
  return n == 0 && y > 0.f ? 1 : n;
}

// Four e3m5 codes of a word: code << 18 is a float's exponent and mantissa, 2^-131 of the code's value, its least codes as
// subnormal floats; the unit, with 2^31 of that, follows 2^100.
__device__ __forceinline__ float v_unit_of(int exp) {
  return exp == 255 ? __uint_as_float(0x7fc00000u) : exp_bits(exp + 31 - V_BIAS + 127 < 254 ? exp + 31 - V_BIAS + 127 : 254);
}
__device__ __forceinline__ float decode_v(unsigned word, int j, float unit) {
  const unsigned bits = (j == 0 ? word << 18 : j == 1 ? word << 10 : j == 2 ? word << 2 : word >> 6) & 0x03fc0000u;
  return __uint_as_float(bits) * 0x1p100f * unit;
}

// A wave's maximum, in a scalar register: within each row of 16 lanes by the vector unit's crossbar, then the four rows.
template <int CTRL>
__device__ __forceinline__ unsigned crossed(unsigned v) {
  return (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
  v = max(v, crossed<0xB1>(v));   // lane ^ 1
  v = max(v, crossed<0x4E>(v));   // lane ^ 2
  v = max(v, crossed<0x141>(v));  // mirrored within 8
  v = max(v, crossed<0x140>(v));  // mirrored within 16
  unsigned m = (unsigned)__builtin_amdgcn_readlane((int)v, 0);
  m = max(m, (unsigned)__builtin_amdgcn_readlane((int)v, 16));
  m = max(m, (unsigned)__builtin_amdgcn_readlane((int)v, 32));
  return max(m, (unsigned)__builtin_amdgcn_readlane((int)v, 48));
}

// A workgroup's elements of tensor t from `base` on (this lane's first). WHOLE: the tensor holds the whole chunk.
template <bool BYTES, bool WHOLE>
__device__ __forceinline__ void adamw_chunk(const AdamArgs& a, const AdamTensor& t, const kg_adamw_values_t& h, long long base) {
  const int lane = threadIdx.x & 63;
  const float decay = (float)(1.0 - (double)h.lr * (double)t.weight_decay);
  const void* weights = t.master ? (const void*)t.master : t.param;
  const int wtype = t.master ? PREC_F32 : t.param_type;
  const long long state0 = t.first_block * kBlock;
  const unsigned high = BYTES ? mix32(h.seed) : 0;

  floatx4 p[kUnroll], g[kUnroll], m[kUnroll], v[kUnroll];
  unsigned mc[kUnroll], vc[kUnroll], me[kUnroll], ve[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const long long i = base + u * kBlock;
    if (!WHOLE && i - lane * 4 >= t.elements) break;  // (whole blocks: uniform over the wave)
    p[u] = load4<WHOLE>(weights, wtype, i, t.elements);
    g[u] = load4<WHOLE>(t.grad, t.grad_type, i, t.elements);
    if constexpr (BYTES) {
      mc[u] = *(const u32_any*)((const unsigned char*)a.m + state0 + i);
      vc[u] = *(const u32_any*)((const unsigned char*)a.v + state0 + i);
      me[u] = a.m_exp[(state0 + i) / kBlock];
      ve[u] = a.v_exp[(state0 + i) / kBlock];
    } else {
      m[u] = __builtin_nontemporal_load((const f32x4_any*)((const float*)a.m + state0 + i));
      v[u] = __builtin_nontemporal_load((const f32x4_any*)((const float*)a.v + state0 + i));
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; u++) {
    const long long i = base + u * kBlock;
    if (!WHOLE && i - lane * 4 >= t.elements) break;
    if constexpr (BYTES) {
      const float mu = unit_of(me[u], M_BIAS), vu = v_unit_of(ve[u]);
      m[u] = floatx4{__builtin_amdgcn_cvt_f32_fp8(mc[u], 0), __builtin_amdgcn_cvt_f32_fp8(mc[u], 1),
                     __builtin_amdgcn_cvt_f32_fp8(mc[u], 2), __builtin_amdgcn_cvt_f32_fp8(mc[u], 3)};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        m[u][j] *= mu;
        const float r = decode_v(vc[u], j, vu);
        v[u][j] = r * r;
      }
    }
    unsigned mtop = 0, vtop = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float gj = g[u][j] * h.grad_scale;
      m[u][j] = m[u][j] * h.beta1 + gj * h.beta1_rest;
      v[u][j] = v[u][j] * h.beta2 + gj * gj * h.beta2_rest;
      if (!WHOLE && i + j >= t.elements) m[u][j] = v[u][j] = 0.f;
    }
    const floatx4 root = roots_of(v[u]);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      // (The quotient by the hardware's reciprocal: an ulp of the update, where the parameter keeps an ulp of itself.)
      p[u][j] = p[u][j] * decay - h.step_size * m[u][j] * __builtin_amdgcn_rcpf(root[j] * h.root_scale + h.eps);
      mtop = max(mtop, __float_as_uint(m[u][j]) & 0x7fffffffu);
      vtop = max(vtop, __float_as_uint(root[j]) & 0x7fffffffu);
    }
    if (t.master) store4_any<WHOLE>(t.master, PREC_F32, i, t.elements, p[u]);
    store4_any<WHOLE>(t.param, t.param_type, i, t.elements, p[u]);
    if constexpr (BYTES) {
      const int em = exp_of(wave_max(mtop), M_CARRY, M_LEAST), ev = exp_of(wave_max(vtop), V_CARRY, V_LEAST);
      const float ms = exp_bits(127 + M_BIAS - (em > 254 ? 254 : em)), vs = exp_bits(127 + V_BIAS - (ev > 254 ? 254 : ev));
      const unsigned long long at = (unsigned long long)(state0 + i);
      const unsigned place = mix32((unsigned)(at >> 32) + high);
      unsigned r[4], cm[4], cv[4];
      float ym[4], yv[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        r[j] = mix32((unsigned)at + j + place);
        ym[j] = fabsf(m[u][j]) * ms;
        yv[j] = root[j] * vs;
        cm[j] = encode_m_normal(ym[j], r[j] & 0xffff);
        cv[j] = encode_v_normal(yv[j], r[j] >> 16);
      }
      // (Few blocks hold a moment so small; a lane that has one takes this for all its four.)
      if (!(fminf(fminf(ym[0], ym[1]), fminf(ym[2], ym[3])) >= 0x1p-6f)) {
#pragma unroll
        for (int j = 0; j < 4; j++) cm[j] = ym[j] >= 0x1p-6f ? cm[j] : encode_m_low(ym[j], r[j] & 0xffff);
      }
      if (!(fminf(fminf(yv[0], yv[1]), fminf(yv[2], yv[3])) >= 32.f)) {
#pragma unroll
        for (int j = 0; j < 4; j++) cv[j] = yv[j] >= 32.f ? cv[j] : encode_v_low(yv[j], r[j] >> 16);
      }
      unsigned mw = 0, vw = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        mw |= ((cm[j] & 0x7f) | ((__float_as_uint(m[u][j]) >> 24) & 0x80)) << (8 * j);
        vw |= (cv[j] & 0xff) << (8 * j);
      }
      *(u32_any*)((unsigned char*)a.m + at) = mw;
      *(u32_any*)((unsigned char*)a.v + at) = vw;
      if (lane == 0) {
        a.m_exp[at / kBlock] = (unsigned char)em;
        a.v_exp[at / kBlock] = (unsigned char)ev;
      }
    } else {
      __builtin_nontemporal_store((f32x4_any)m[u], (f32x4_any*)((float*)a.m + state0 + i));
      __builtin_nontemporal_store((f32x4_any)v[u], (f32x4_any*)((float*)a.v + state0 + i));
    }
  }
}

template <bool BYTES>
__global__ __launch_bounds__(kWaves * 64) void adamw_kernel(AdamArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wg = blockIdx.x;
  // The tensor of this workgroup: the last one that starts at or before it.
  int ti = __popcll(__ballot(a.start[lane] <= wg));
  ti += __popcll(__ballot(lane < kTensors - 64 && a.start[64 + (lane < kTensors - 64 ? lane : 0)] <= wg));
  ti = __builtin_amdgcn_readfirstlane(ti) - 1;
  const AdamTensor t = a.t[ti].open();
  const kg_adamw_values_t h = a.device_values ? *a.device_values : a.values;
  const long long first = (long long)(wg - a.start[ti]) * kChunk, base = first + (wave * kUnroll) * kBlock + lane * 4;
  if (first + kChunk <= t.elements) adamw_chunk<BYTES, true>(a, t, h, base);
  else adamw_chunk<BYTES, false>(a, t, h, base);
}

// kUnroll blocks a wave, four elements of each a lane, all loads before the first store: 240 M moments of 8 bits to bf16 in 220 us
// (6.5 TB/s; one block a wave: 305).
template <bool BYTES>
__global__ __launch_bounds__(kWaves * 64) void adamw_moments_kernel(const void* m, const void* v, const unsigned char* m_exp,
                                                                    const unsigned char* v_exp, long long blocks, int type,
                                                                    void* out_m, void* out_root) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (long long b0 = ((long long)blockIdx.x * kWaves + wave) * kUnroll; b0 < blocks; b0 += (long long)gridDim.x * kWaves * kUnroll) {
    unsigned mc[kUnroll], vc[kUnroll], me[kUnroll], ve[kUnroll];
    floatx4 fm[kUnroll], fr[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
      const long long b = b0 + u < blocks ? b0 + u : blocks - 1, i = b * kBlock + lane * 4;
      if constexpr (BYTES) {
        mc[u] = __builtin_nontemporal_load((const u32_any*)((const unsigned char*)m + i));
        vc[u] = __builtin_nontemporal_load((const u32_any*)((const unsigned char*)v + i));
        me[u] = m_exp[b];
        ve[u] = v_exp[b];
      } else {
        fm[u] = __builtin_nontemporal_load((const f32x4_any*)((const float*)m + i));
        fr[u] = __builtin_nontemporal_load((const f32x4_any*)((const float*)v + i));
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
      if (b0 + u >= blocks) break;
      if constexpr (BYTES) {
        const float mu = unit_of(me[u], M_BIAS), vu = v_unit_of(ve[u]);
        fm[u] = floatx4{__builtin_amdgcn_cvt_f32_fp8(mc[u], 0), __builtin_amdgcn_cvt_f32_fp8(mc[u], 1),
                        __builtin_amdgcn_cvt_f32_fp8(mc[u], 2), __builtin_amdgcn_cvt_f32_fp8(mc[u], 3)} * mu;
#pragma unroll
        for (int j = 0; j < 4; j++) fr[u][j] = decode_v(vc[u], j, vu);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) fr[u][j] = sqrtf(fr[u][j]);
      }
      const long long i = (b0 + u) * kBlock + lane * 4;
      store4_any<true>(out_m, type, i, blocks * kBlock, fm[u]);
      store4_any<true>(out_root, type, i, blocks * kBlock, fr[u]);
    }
  }
}

}  // namespace

void launch_adamw(int count, const kg_adamw_tensor* tensors, const kg_adamw_state& state, const kg_adamw_values_t& values,
                  const kg_adamw_values_t* device_values, hipStream_t s) {
  AdamArgs a;
  a.values = values;
  a.device_values = device_values;
  a.m = state.m; a.v = state.v;
  a.m_exp = state.m_exp; a.v_exp = state.v_exp;
  int n = 0;
  long long groups = 0;
  auto flush = [&] {
    if (!n) return;
    for (int i = n; i < kTensors; i++) a.start[i] = INT_MAX;
    if (state.state_bits == 8) launch_k(adamw_kernel<true>, dim3((unsigned)groups), kWaves * 64, 0, s, a);
    else launch_k(adamw_kernel<false>, dim3((unsigned)groups), kWaves * 64, 0, s, a);
    KGX_CHECK_LAUNCH();
    n = 0;
    groups = 0;
  };
  for (int i = 0; i < count; i++) {
    const kg_adamw_tensor& t = tensors[i];
    // (A launch takes up to 2^22 workgroups, 2^34 elements: a larger tensor goes in pieces of whole blocks.)
    constexpr long long most = 1ll << 22;
    for (long long done = 0; done < t.elements;) {
      if (n == kTensors || groups == most) flush();
      const long long left = t.elements - done, room = (most - groups) * kChunk, take = left < room ? left : room;
      AdamTensor d;
      const long long ps = t.param_type == PREC_F32 ? 4 : 2, gs = t.grad_type == PREC_F32 ? 4 : 2;
      d.param = (char*)t.param + done * ps;
      d.grad = (const char*)t.grad + done * gs;
      d.master = t.master ? t.master + done : nullptr;
      d.elements = take;
      d.first_block = t.first_block + done / kBlock;
      d.weight_decay = (float)t.weight_decay;
      d.param_type = (short)t.param_type;
      d.grad_type = (short)t.grad_type;
      if (((unsigned long long)d.param | (unsigned long long)d.grad | (unsigned long long)d.master) >> 48)
        throw std::runtime_error("kgx AdamW: an address is over 48 bits");
      a.t[n] = AdamPacked::of(d);
      a.start[n++] = (int)groups;
      groups += (take + kChunk - 1) / kChunk;
      done += take;
    }
  }
  flush();
}

void launch_adamw_moments(long long blocks, const kg_adamw_state& state, int type, void* m, void* root, hipStream_t s) {
  if (blocks <= 0) return;
  const long long groups = (blocks + kWaves * kUnroll - 1) / (kWaves * kUnroll);
  const dim3 grid((unsigned)(groups < (1 << 20) ? groups : (1 << 20)));
  if (state.state_bits == 8)
    launch_k(adamw_moments_kernel<true>, grid, kWaves * 64, 0, s, state.m, state.v, state.m_exp, state.v_exp, blocks, type, m, root);
  else
    launch_k(adamw_moments_kernel<false>, grid, kWaves * 64, 0, s, state.m, state.v, state.m_exp, state.v_exp, blocks, type, m, root);
  KGX_CHECK_LAUNCH();
}

}  // namespace kgx
