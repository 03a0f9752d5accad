// The angle of a rotary position, as all kernels that turn pairs work it out.
#pragma once
#include <hip/hip_runtime.h>

namespace tracea_amd {

// The angle is formed and reduced in 64 bits: the product of a 31-bit position and a 24-bit frequency has up to 55 bits,
// and what counts is its remainder of a whole turn.  32 bits would be off by 2^-24 of the ANGLE: 0.004 rad at position 65536.
// The sine and cosine of the remainder are fp32.  A position is a whole number of 32 bits, with a sign or (a place in a sequence) without.
__device__ __forceinline__ void turn(double position, float freq, float sign, float &c, float &s) {
  const double turns = position * (double)freq * 0.15915494309189535;
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  s *= sign;
}

}  // namespace tracea_amd
