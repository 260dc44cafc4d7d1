// The 8-bit form of a saved activation: each run of 32 values along a row (the last one may be shorter) shares a power
// of two 2^e, kept as the byte e + 127; a value is kept as e4m3(v / 2^e), rounded once to nearest even.
// 2^e is the smallest power of two, at least 2^-126, with which no finite value of the run passes 448 (the largest
// e4m3 number), so nothing is clipped; dividing by it is exact.  Values that are not finite become NaN and do not
// count for the scale.
#pragma once
#include "common.h"

constexpr int kAct8Group = 32;

// scale byte for the largest finite magnitude of a run, given as its f32 bit pattern
__device__ __forceinline__ int act8_scale_byte(uint32_t most) {
    // 448 = 1.75 * 2^8: one power more where the significand is above 1.75, that is where adding 2^21 - 1 carries
    const int b = (int)((most + 0x1fffffu) >> 23) - 8;
    return b < 1 ? 1 : b;
}
__device__ __forceinline__ float act8_inverse(int byte) { return __builtin_bit_cast(float, (uint32_t)(254 - byte) << 23); }
// 2^(byte - 127); byte 0 is a subnormal f32, 255 stands for NaN
__device__ __forceinline__ float act8_scale(uint32_t byte) {
    return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}
