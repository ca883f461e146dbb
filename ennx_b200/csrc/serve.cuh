// serve.cuh -- device helpers shared by the serving operators (packed-prompt
// and single-token attention, few-token MoE, few-token packed products).
#pragma once

#include "common.cuh"

namespace ennx {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rotary table in turns: angle of pair i at position p is 2*pi * p * inv[i].
// Positions reach 10^5 and more, where a 32-bit product has lost the angle, so
// p * inv[i] is formed and reduced to [-1/2, 1/2] in 64 bits; only the reduced
// turn is rounded to 32 (error 2^-25 turns, 2e-7 radians).
struct RopeTable {
  double inv[64];
};
__device__ __forceinline__ void rope_sincos(const RopeTable& t, int i, int pos, float* s, float* c) {
  const double turns = (double)pos * t.inv[i];
  sincospif((float)(2.0 * (turns - rint(turns))), s, c);
}
// host: inv[i] = theta^(-2i/128) / (2*pi)
const RopeTable& rope_table(float theta);

}  // namespace ennx
