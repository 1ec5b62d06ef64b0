// Cosine and sine of a position's angle, shared by the kernels of rotary positions with frequencies in turns.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace cb200 {

// The angle is found modulo one turn in 64-bit binary fractions: position * turns in integers drops whole turns exactly, so that a
// position of a million has an angle as good as position 1 (in 32-bit floats it would be off by 0.06 rad). The fraction's nearest quarter
// turn is split off as an integer too; what is left lies in [-1/4, 1/4) half turns and keeps 2^-26 of a turn in a float.
__device__ __forceinline__ float2 turn_cos_sin(uint64_t turns, int position, float factor) {
  const uint64_t f = turns * static_cast<uint64_t>(static_cast<long long>(position));
  const uint64_t quarter = (f + (1ull << 61)) >> 62;
  const long long rest = static_cast<long long>(f - (quarter << 62));
  float s, c;
  sincospif(static_cast<float>(rest) * 1.0842021724855044e-19f, &s, &c);       // 2^-63: rest in half turns
  const float2 r = (quarter & 1) ? make_float2(-s, c) : make_float2(c, s);
  return (quarter & 2) ? make_float2(-r.x * factor, -r.y * factor) : make_float2(r.x * factor, r.y * factor);
}

}  // namespace cb200
