// Rotary positions: the angle of a (position, frequency) pair and the turn of a pair of features.
// Shared by the rotary kernel and by the epilogue of the 4-bit products.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace mkb {

struct RotaryArgs {
  const void* positions;   // int32 or int64, one per token
  int pos64;
  const float* inv_freq;   // radians per position, one per pair of features
  float scale;             // multiplies cos and sin
};

__device__ __forceinline__ long long rotary_position(const RotaryArgs& a, long long token) {
  return a.pos64 ? static_cast<const long long*>(a.positions)[token]
                 : static_cast<const int*>(a.positions)[token];
}

// cos and sin of position * inv_freq, times scale.  In turns (1/2pi radians) the whole part can be
// dropped exactly; the product is taken in 64 bits, because at position 1e6 an fp32 product has
// lost 0.03 radians before the cosine is taken.  What is left of it (below half a turn) fits fp32.
__device__ __forceinline__ float2 rotary_cos_sin(long long position, float inv_freq, float scale) {
  double turns = (double)position * ((double)inv_freq * 0.15915494309189535);
  turns -= rint(turns);
  float s, c;
  sincospif(2.0f * (float)turns, &s, &c);
  return make_float2(c * scale, s * scale);
}

// (x, y) turned by the angle whose cosine and sine are cs.
__device__ __forceinline__ float2 rotary_turn(float x, float y, float2 cs) {
  return make_float2(x * cs.x - y * cs.y, y * cs.x + x * cs.y);
}

}  // namespace mkb
