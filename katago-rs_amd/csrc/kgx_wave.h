// Exchanges within a wave on the vector unit's crossbar, without LDS.
#pragma once
#include <hip/hip_runtime.h>

namespace kgx {

template <int CTRL>
__device__ __forceinline__ float crossed(float v) {
  return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_of(float v, int lane) {
  return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}
// A wave's sum or maximum, in every lane: within each row of 16 lanes by the lanes' crossbar of the vector unit, then the four
// rows through scalar registers (six exchanges through LDS, before, were most of a narrow row's time). Every lane is active.
template <bool MAX>
__device__ __forceinline__ float wave_reduce(float v) {
  auto join = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
  v = join(v, crossed<0xB1>(v));   // lane ^ 1
  v = join(v, crossed<0x4E>(v));   // lane ^ 2
  v = join(v, crossed<0x141>(v));  // mirrored within 8
  v = join(v, crossed<0x140>(v));  // mirrored within 16
  return join(join(lane_of(v, 0), lane_of(v, 16)), join(lane_of(v, 32), lane_of(v, 48)));
}
// The same sum over each `share` neighbouring lanes (a power of two up to 64, the same for the wave).
__device__ __forceinline__ float share_sum(float v, int share) {
  if (share > 1) v += crossed<0xB1>(v);
  if (share > 2) v += crossed<0x4E>(v);
  if (share > 4) v += crossed<0x141>(v);
  if (share > 8) v += crossed<0x140>(v);
  if (share > 16) {
    const float low = lane_of(v, 0) + lane_of(v, 16), high = lane_of(v, 32) + lane_of(v, 48);
    v = share == 64 ? low + high : threadIdx.x & 32 ? high : low;
  }
  return v;
}

}  // namespace kgx
