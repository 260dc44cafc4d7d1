// Loads and stores of VEC neighbouring elements of a row as f32 values, for kernels whose rows may be f32 or bf16.
// VEC > 1 needs the address aligned to VEC elements; bf16 stores round to nearest even.
#pragma once
#include "common.h"

template <typename T, int VEC>
__device__ __forceinline__ void tc_load_row(const T *p, float (&v)[VEC]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (VEC == 8) {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        } else if constexpr (VEC == 4) {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = a[j];
        } else {
            static_assert(VEC == 1, "1, 4 or 8 elements");
            v[0] = *p;
        }
    } else {
        if constexpr (VEC == 8) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[2 * j] = tc_bf16_lo(w[j]); v[2 * j + 1] = tc_bf16_hi(w[j]); }
        } else if constexpr (VEC == 4) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(p);
#pragma unroll
            for (int j = 0; j < 2; ++j) { v[2 * j] = tc_bf16_lo(w[j]); v[2 * j + 1] = tc_bf16_hi(w[j]); }
        } else {
            static_assert(VEC == 1, "1, 4 or 8 elements");
            v[0] = tc_bf16_lo(*p);
        }
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void tc_store_row(T *p, const float (&v)[VEC]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (VEC == 1) {
            p[0] = v[0];
        } else {
#pragma unroll
            for (int k = 0; k < VEC; k += 4) *reinterpret_cast<f32x4 *>(p + k) = f32x4{v[k], v[k + 1], v[k + 2], v[k + 3]};
        }
    } else {
        if constexpr (VEC == 8) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = tc_pack_bf16(v[2 * j], v[2 * j + 1]);
            *reinterpret_cast<u32x4 *>(p) = w;
        } else if constexpr (VEC == 4) {
            *reinterpret_cast<u32x2 *>(p) = u32x2{tc_pack_bf16(v[0], v[1]), tc_pack_bf16(v[2], v[3])};
        } else {
            *p = __builtin_bit_cast(uint16_t, (__bf16)v[0]);
        }
    }
}

// whether a row-major operand can be read or written VEC elements at a time
static inline bool tc_rows_aligned(const void *p, long ld, int esz, int vec) {
    return ((uintptr_t)p % ((size_t)esz * vec)) == 0 && ld % vec == 0;
}
