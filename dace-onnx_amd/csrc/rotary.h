// The angle that a pair of a head is turned by.
#pragma once

#include "common.h"

namespace mi355x {

constexpr int ROTARY_MAX_AXES = 8, ROTARY_LDS_ANGLES = 2048;

// Cosine and sine of position * frequency. The product is taken in float64: exact for positions below 2^29, rounded from there on. It is counted in turns, by a rounded
// factor, and brought into one turn there: off by less than 2^-51 of the turns in all (position 2^40 at frequency 1: 5e-4 radians). Positions far into a context
// are thousands of turns, of which float32 would leave few right digits (position 100000: 0.004 radians). What is left is rounded to float32, pi 2^-24 of an angle at most, and its
// cosine and sine are float32: float32 results are off by 4.9e-8 in the 2-norm, where cosine and sine taken in float64 give 3.6e-8.
__device__ __forceinline__ float2 rotary_turn(int64_t position, float frequency) {
    const double turns = (double)position * (double)frequency * 0.15915494309189533577;
    float sine, cosine;
    sincospif((float)(2.0 * (turns - rint(turns))), &sine, &cosine);
    return make_float2(cosine, sine);
}

}  // namespace mi355x
