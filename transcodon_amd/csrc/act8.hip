// 8-bit activation checkpoints: packing, unpacking, and GELU with its gradient through a checkpoint of its input.
//
//   tc_act8_pack     x -> codes, scales
//   tc_gelu_act8     u -> gelu(u), codes and scales of u                        (forward)
//   tc_dgelu_act8    dy, codes, scales -> dy * gelu'(u8), gelu(u8) again        (backward; u8: what the codes stand for)
//
// A lane owns 8 neighbouring values of a row, four lanes a run of 32; rows that do not fit (width or alignment) go one
// value a lane, 32 lanes a run.  Everything is one pass over memory.
#include "act8.h"
#include "row_io.h"

namespace {

// Phi(x) and exp(-x^2 / 2).  With a = |x| the lower tail is Phi(-a) = exp(-a^2 / 2) t P(t), t = 1 / (1 + 0.3 a): P is a
// polynomial of degree 7 fitted to exp(a^2 / 2) Phi(-a) / t over a in [0, 14] for the least relative error (1.5e-7).
// The tail keeps its relative accuracy, which 1 + erf(x / sqrt 2) loses, and the exponential serves the derivative too.
__device__ __forceinline__ float normal_cdf(float x, float &e) {
    const float a = fabsf(x);
    const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.3f, 1.0f));
    e = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);       // -log2(e) / 2
    float q = 0.03567494824528694f;
    q = fmaf(q, t, -0.1572037637233734f);
    q = fmaf(q, t, 0.20635460317134857f);
    q = fmaf(q, t, -0.053684573620557785f);
    q = fmaf(q, t, 0.1285620778799057f);
    q = fmaf(q, t, 0.09991336613893509f);
    q = fmaf(q, t, 0.12075397372245789f);
    q = fmaf(q, t, 0.11962930113077164f);
    q *= t * e;
    return x < 0.f ? q : 1.0f - q;
}

struct Act8Params {
    const void *x;           // u, x or dy
    long ldx;
    void *y;                 // act, du or the unpacked values; dense
    void *again;             // gelu of the checkpoint (may be null)
    uint8_t *codes, *scales;
    long n_pieces;           // rows * pieces per row
    int E, groups, pieces;   // width, runs per row, pieces (of VEC values) per row
};

// largest magnitude bits over the lanes of a run
template <int VEC>
__device__ __forceinline__ uint32_t run_max(uint32_t m) {
    if constexpr (VEC == 8) {
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));     // lane ^ 1
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));     // lane ^ 2
    } else {
#pragma unroll
        for (int off = 1; off < kAct8Group; off <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
    }
    return m;
}

template <int VEC>
__device__ __forceinline__ void store_codes(uint8_t *dst, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        u32x2 w;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k], v[4 * k + 1], 0, false);
            c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2], v[4 * k + 3], c, true);
            w[k] = (uint32_t)c;
        }
        *reinterpret_cast<u32x2 *>(dst) = w;
    } else {
        *dst = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[0], 0, false);
    }
}

template <int VEC>
__device__ __forceinline__ void load_codes(const uint8_t *src, float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(src);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], true);
            v[4 * k] = lo[0]; v[4 * k + 1] = lo[1]; v[4 * k + 2] = hi[0]; v[4 * k + 3] = hi[1];
        }
    } else {
        v[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)*src, false)[0];
    }
}

// T: type of x and y.  FLAT: rows follow each other without a gap and hold whole runs, so a piece's place is its number.
template <typename T, int VEC, bool FLAT, bool GELU>
__global__ __launch_bounds__(256) void act8_pack_kernel(const Act8Params p) {
    constexpr int LPG = kAct8Group / VEC;                         // lanes per run
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < p.n_pieces; i += (long)gridDim.x * 256) {
        long row = 0, at_x, at;
        int col = 0;
        bool in = true;
        if constexpr (FLAT) {
            at_x = at = i * VEC;
        } else {
            row = i / p.pieces;
            col = (int)(i - row * p.pieces) * VEC;
            in = col < p.E;
            at_x = row * p.ldx + col;
            at = row * p.E + col;
        }
        float v[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 0.f;
        if (in) tc_load_row<T, VEC>(static_cast<const T *>(p.x) + at_x, v);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = max(m, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
        m = run_max<VEC>(m);
        float w[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] = v[j];
        if (m >= 0x7f800000u) {                                    // some value is not finite (the whole run comes here)
            m = 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const uint32_t b = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
                if (b < 0x7f800000u) m = max(m, b);
                else w[j] = __builtin_nanf("");
            }
            m = run_max<VEC>(m);
        }
        const int byte = act8_scale_byte(m);
        const float inv = act8_inverse(byte);
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] *= inv;
        if (in) {
            store_codes<VEC>(p.codes + at, w);
            if constexpr (GELU) {
                float e;
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] *= normal_cdf(v[j], e);
                tc_store_row<T, VEC>(static_cast<T *>(p.y) + at, v);
            }
        }
        if ((threadIdx.x & (LPG - 1)) == 0) p.scales[FLAT ? i / LPG : row * p.groups + col / kAct8Group] = (uint8_t)byte;
    }
}

// GELU: x is dy, y is du; otherwise y receives the values that the codes stand for
template <typename T, int VEC, bool FLAT, bool GELU>
__global__ __launch_bounds__(256) void act8_read_kernel(const Act8Params p) {
    constexpr int LPG = kAct8Group / VEC;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < p.n_pieces; i += (long)gridDim.x * 256) {
        long row = 0, at_x, at;
        int col = 0;
        if constexpr (FLAT) {
            at_x = at = i * VEC;
        } else {
            row = i / p.pieces;
            col = (int)(i - row * p.pieces) * VEC;
            if (col >= p.E) continue;
            at_x = row * p.ldx + col;
            at = row * p.E + col;
        }
        float v[VEC], d[VEC];
        load_codes<VEC>(p.codes + at, v);
        const float scale = act8_scale(p.scales[FLAT ? i / LPG : row * p.groups + col / kAct8Group]);
        if constexpr (GELU) tc_load_row<T, VEC>(static_cast<const T *>(p.x) + at_x, d);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] *= scale;
        if constexpr (GELU) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float e;
                const float cdf = normal_cdf(v[j], e);
                d[j] *= fmaf(v[j] * 0.3989422804014327f, e, cdf);  // Phi(u) + u phi(u)
                v[j] *= cdf;
            }
            tc_store_row<T, VEC>(static_cast<T *>(p.y) + at, d);
            if (p.again) tc_store_row<T, VEC>(static_cast<T *>(p.again) + at, v);
        } else {
            tc_store_row<T, VEC>(static_cast<T *>(p.y) + at, v);
        }
    }
}

int act8_check(const char *who, int dtype, long M, int E) {
    TC_REQUIRE(dtype == TC_F32 || dtype == TC_BF16, "%s: bad dtype %d", who, dtype);
    TC_REQUIRE(M > 0 && M <= 0x7fffffffL && E > 0 && E <= (1 << 20), "%s: bad shape M=%ld E=%d", who, M, E);
    return TC_OK;
}

Act8Params act8_params(const void *x, long ldx, void *y, void *again, void *codes, void *scales, long M, int E, int esz, bool &vec,
                       bool &flat) {
    Act8Params p{};
    p.x = x; p.ldx = ldx; p.y = y; p.again = again;
    p.codes = static_cast<uint8_t *>(codes);
    p.scales = static_cast<uint8_t *>(scales);
    p.E = E;
    p.groups = (E + kAct8Group - 1) / kAct8Group;
    vec = E % 8 == 0 && (!x || tc_rows_aligned(x, ldx, esz, 8)) && (!y || tc_rows_aligned(y, E, esz, 8)) &&
          (!again || tc_rows_aligned(again, E, esz, 8)) && (uintptr_t)codes % 8 == 0;
    flat = E % kAct8Group == 0 && (!x || ldx == E);
    p.pieces = p.groups * (kAct8Group / (vec ? 8 : 1));
    p.n_pieces = M * p.pieces;
    return p;
}

dim3 act8_grid(const Act8Params &p) {
    const long blocks = (p.n_pieces + 255) / 256, most = 1L << 20;      // a launch holds fewer than 2^32 threads
    return dim3((unsigned)(blocks < most ? blocks : most));
}

#define TC_A8(KERNEL, T, GELU)                                                                                          \
    do {                                                                                                                \
        if (vec && flat) TC_LAUNCH((KERNEL<T, 8, true, GELU>), act8_grid(p), dim3(256), 0, s, p);                       \
        else if (vec) TC_LAUNCH((KERNEL<T, 8, false, GELU>), act8_grid(p), dim3(256), 0, s, p);                         \
        else TC_LAUNCH((KERNEL<T, 1, false, GELU>), act8_grid(p), dim3(256), 0, s, p);                                  \
    } while (0)

int pack_call(const char *who, int dtype, const void *x, long ldx, void *act, void *codes, void *scales, long M, int E, bool gelu,
              void *stream) {
    const int rc = act8_check(who, dtype, M, E);
    if (rc != TC_OK) return rc;
    const int esz = dtype == TC_BF16 ? 2 : 4;
    TC_REQUIRE(x && codes && scales && (act || !gelu), "%s: null operand", who);
    TC_REQUIRE(ldx >= E && ((uintptr_t)x | (uintptr_t)act) % esz == 0, "%s: bad row stride or alignment", who);
    hipStream_t s = static_cast<hipStream_t>(stream);
    bool vec, flat;
    const Act8Params p = act8_params(x, ldx, act, nullptr, codes, scales, M, E, esz, vec, flat);
    if (dtype == TC_F32) {
        if (gelu) TC_A8(act8_pack_kernel, float, true); else TC_A8(act8_pack_kernel, float, false);
    } else {
        if (gelu) TC_A8(act8_pack_kernel, uint16_t, true); else TC_A8(act8_pack_kernel, uint16_t, false);
    }
    TC_CHECK_LAUNCH(who);
    return TC_OK;
}

}  // namespace

extern "C" int tc_act8_pack(int dtype, const void *x, long ldx, void *codes, void *scales, long M, int E, void *stream) {
    return pack_call("tc_act8_pack", dtype, x, ldx, nullptr, codes, scales, M, E, false, stream);
}

extern "C" int tc_gelu_act8(int dtype, const void *u, long ldu, void *act, void *codes, void *scales, long M, int E, void *stream) {
    return pack_call("tc_gelu_act8", dtype, u, ldu, act, codes, scales, M, E, true, stream);
}

extern "C" int tc_act8_unpack(int dtype, const void *codes, const void *scales, void *out, long M, int E, void *stream) {
    const int rc = act8_check("tc_act8_unpack", dtype, M, E);
    if (rc != TC_OK) return rc;
    const int esz = dtype == TC_BF16 ? 2 : 4;
    TC_REQUIRE(codes && scales && out && (uintptr_t)out % esz == 0, "tc_act8_unpack: null or misaligned operand");
    hipStream_t s = static_cast<hipStream_t>(stream);
    bool vec, flat;
    const Act8Params p = act8_params(nullptr, 0, out, nullptr, const_cast<void *>(codes), const_cast<void *>(scales), M, E, esz, vec, flat);
    if (dtype == TC_F32) TC_A8(act8_read_kernel, float, false);
    else TC_A8(act8_read_kernel, uint16_t, false);
    TC_CHECK_LAUNCH("tc_act8_unpack");
    return TC_OK;
}

extern "C" int tc_dgelu_act8(int dtype, const void *dy, long ld_dy, const void *codes, const void *scales, void *du, void *act, long M,
                             int E, void *stream) {
    const int rc = act8_check("tc_dgelu_act8", dtype, M, E);
    if (rc != TC_OK) return rc;
    const int esz = dtype == TC_BF16 ? 2 : 4;
    TC_REQUIRE(dy && codes && scales && du, "tc_dgelu_act8: null operand");
    TC_REQUIRE(ld_dy >= E && ((uintptr_t)dy | (uintptr_t)du | (uintptr_t)act) % esz == 0, "tc_dgelu_act8: bad row stride or alignment");
    hipStream_t s = static_cast<hipStream_t>(stream);
    bool vec, flat;
    const Act8Params p = act8_params(dy, ld_dy, du, act, const_cast<void *>(codes), const_cast<void *>(scales), M, E, esz, vec, flat);
    if (dtype == TC_F32) TC_A8(act8_read_kernel, float, true);
    else TC_A8(act8_read_kernel, uint16_t, true);
    TC_CHECK_LAUNCH("tc_dgelu_act8");
    return TC_OK;
}
