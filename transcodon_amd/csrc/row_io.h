// Loads and stores of VEC neighbouring elements of a row as f32 values, for kernels whose rows may be f32 or bf16; bf16
// stores round to nearest even.
#pragma once
#include "common.h"
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) uint32_t u32x8;

// what a load of VEC elements leaves in registers, before it is widened to f32
template <typename T, int VEC>
struct TcRaw {
    typedef typename std::conditional<sizeof(T) * VEC == 2, uint16_t,
            typename std::conditional<sizeof(T) * VEC == 4, uint32_t,
            typename std::conditional<sizeof(T) * VEC == 8, u32x2,
            typename std::conditional<sizeof(T) * VEC == 16, u32x4, u32x8>::type>::type>::type>::type type;
};
// LOOSE: p is aligned to its element only (gfx950 takes such vector loads) and n elements are there; those past them read as 0
template <typename T, int VEC, bool LOOSE = false>
__device__ __forceinline__ typename TcRaw<T, VEC>::type tc_raw_load(const T *p, int n = VEC) {
    typename TcRaw<T, VEC>::type raw;
    if constexpr (!LOOSE) {
        raw = *reinterpret_cast<const typename TcRaw<T, VEC>::type *>(p);
    } else if (n >= VEC) {
        __builtin_memcpy(&raw, p, sizeof(raw));
    } else {
        T e[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[j] = j < n ? p[j] : T{};
        __builtin_memcpy(&raw, e, sizeof(raw));
    }
    return raw;
}
template <typename T, int VEC>
__device__ __forceinline__ void tc_raw_widen(const typename TcRaw<T, VEC>::type &raw, float (&v)[VEC]) {
    if constexpr (sizeof(T) == 4) {
        __builtin_memcpy(v, &raw, sizeof(v));
    } else if constexpr (VEC == 1) {
        v[0] = tc_bf16_lo(raw);
    } else {
        uint32_t w[VEC / 2];
        __builtin_memcpy(w, &raw, sizeof(w));
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) { v[2 * j] = tc_bf16_lo(w[j]); v[2 * j + 1] = tc_bf16_hi(w[j]); }
    }
}

template <typename T, int VEC, bool LOOSE = false>
__device__ __forceinline__ void tc_load_row(const T *p, float (&v)[VEC], int n = VEC) {
    tc_raw_widen<T, VEC>(tc_raw_load<T, VEC, LOOSE>(p, n), v);
}

template <typename T, int VEC, bool LOOSE = false>
__device__ __forceinline__ void tc_store_row(T *p, const float (&v)[VEC], int n = VEC) {
    typename TcRaw<T, VEC>::type raw;
    if constexpr (sizeof(T) == 4) {
        __builtin_memcpy(&raw, v, sizeof(v));
    } else if constexpr (VEC == 1) {
        raw = __builtin_bit_cast(uint16_t, (__bf16)v[0]);
    } else {
        uint32_t w[VEC / 2];
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) w[j] = tc_pack_bf16(v[2 * j], v[2 * j + 1]);
        __builtin_memcpy(&raw, w, sizeof(w));
    }
    if constexpr (!LOOSE) {
        *reinterpret_cast<typename TcRaw<T, VEC>::type *>(p) = raw;
    } else if (n >= VEC) {
        __builtin_memcpy(p, &raw, sizeof(raw));
    } else {
        T e[VEC];
        __builtin_memcpy(e, &raw, sizeof(raw));
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < n) p[j] = e[j];
    }
}

// whether a row-major operand can be read or written VEC elements at a time with aligned accesses
static inline bool tc_rows_aligned(const void *p, long ld, int esz, int vec) {
    return ((uintptr_t)p % ((size_t)esz * vec)) == 0 && ld % vec == 0;
}
