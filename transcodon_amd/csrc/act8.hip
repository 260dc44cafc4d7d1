// 8-bit activation checkpoints: packing, unpacking, and GELU with its gradient through a checkpoint of its input.
//
//   tc_act8_pack     x -> codes, scales
//   tc_gelu_act8     u -> gelu(u), codes and scales of u                        (forward)
//   tc_dgelu_act8    dy, codes, scales -> dy * gelu'(u8), gelu(u8) again        (backward; u8: what the codes stand for)
//
// A lane owns 8 neighbouring values of a row, four lanes a run of 32.  Where rows follow each other without a gap and hold
// whole runs, a piece's place is its number (FLAT); otherwise lanes are dealt to rows, addresses may be aligned to single
// elements only, and a row's last values go one by one.  Everything is one pass over memory.
#include "act8.h"
#include "row_io.h"

namespace {

// Phi(x) and exp(-x^2 / 2).  With a = |x| the lower tail is Phi(-a) = exp(-a^2 / 2) t P(t), t = 1 / (1 + 0.3 a): P is a
// polynomial of degree 7 fitted to exp(a^2 / 2) Phi(-a) / t over a in [0, 14] for the least relative error (1.7e-7).
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

constexpr int VEC = 8;
constexpr int kLanesPerRun = kAct8Group / VEC;

struct Act8Params {
    const void *x;           // u, x or dy
    long ldx;
    void *y;                 // act, du or the unpacked values; dense
    void *again;             // gelu of the checkpoint (may be null)
    uint8_t *codes, *scales;
    long rows, n_pieces;     // n_pieces (FLAT): rows * E / VEC
    int E, groups;           // width, runs per row
    int lanes_log2;          // not FLAT: lanes of a row, at least those of a run
};

// largest magnitude bits over the lanes of a run
__device__ __forceinline__ uint32_t run_max(uint32_t m) {
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));     // lane ^ 1
    return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));  // lane ^ 2
}

template <bool LOOSE>
__device__ __forceinline__ void store_codes(uint8_t *dst, const float (&v)[VEC], int n) {
    u32x2 w;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k], v[4 * k + 1], 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2], v[4 * k + 3], c, true);
        w[k] = (uint32_t)c;
    }
    if constexpr (!LOOSE) {
        *reinterpret_cast<u32x2 *>(dst) = w;
    } else if (n >= VEC) {
        __builtin_memcpy(dst, &w, VEC);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < n) dst[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    }
}

template <bool LOOSE>
__device__ __forceinline__ void load_codes(const uint8_t *src, float (&v)[VEC], int n) {
    u32x2 w = u32x2{0u, 0u};
    if constexpr (!LOOSE) {
        w = *reinterpret_cast<const u32x2 *>(src);
    } else if (n >= VEC) {
        __builtin_memcpy(&w, src, VEC);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < n) w[j >> 2] |= (uint32_t)src[j] << (8 * (j & 3));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], true);
        v[4 * k] = lo[0]; v[4 * k + 1] = lo[1]; v[4 * k + 2] = hi[0]; v[4 * k + 3] = hi[1];
    }
}

// One piece: x and the dense outputs at at_x and at, n of its values are there (0 .. VEC; all four lanes of a run call this).
template <typename T, bool LOOSE, bool GELU>
__device__ __forceinline__ void pack_piece(const Act8Params &p, long at_x, long at, long run, int n) {
    float v[VEC], w[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = 0.f;
    if (!LOOSE || n > 0) tc_load_row<T, VEC, LOOSE>(static_cast<const T *>(p.x) + at_x, v, n);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        m = max(m, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
        w[j] = v[j];
    }
    m = run_max(m);
    if (m >= 0x7f800000u) {                                    // some value is not finite (the whole run comes here)
        m = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const uint32_t b = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
            if (b < 0x7f800000u) m = max(m, b);
            else w[j] = __builtin_nanf("");
        }
        m = run_max(m);
    }
    const int byte = act8_scale_byte(m);
    const float inv = act8_inverse(byte);
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[j] *= inv;
    if (!LOOSE || n > 0) {
        store_codes<LOOSE>(p.codes + at, w, n);
        if constexpr (GELU) {
            float e;
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] *= normal_cdf(v[j], e);
            tc_store_row<T, VEC, LOOSE>(static_cast<T *>(p.y) + at, v, n);
        }
    }
    if ((threadIdx.x & (kLanesPerRun - 1)) == 0) p.scales[run] = (uint8_t)byte;
}

// GELU: x is dy, y is du; otherwise y receives the values that the codes stand for
template <typename T, bool LOOSE, bool GELU>
__device__ __forceinline__ void read_piece(const Act8Params &p, long at_x, long at, long run, int n) {
    if (LOOSE && n <= 0) return;
    float v[VEC], d[VEC];
    load_codes<LOOSE>(p.codes + at, v, n);
    const float scale = act8_scale(p.scales[run]);
    if constexpr (GELU) tc_load_row<T, VEC, LOOSE>(static_cast<const T *>(p.x) + at_x, d, n);
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
        tc_store_row<T, VEC, LOOSE>(static_cast<T *>(p.y) + at, d, n);
        if (p.again) tc_store_row<T, VEC, LOOSE>(static_cast<T *>(p.again) + at, v, n);
    } else {
        tc_store_row<T, VEC, LOOSE>(static_cast<T *>(p.y) + at, v, n);
    }
}

template <typename T, bool FLAT, bool GELU, bool READ>
__global__ __launch_bounds__(256) void act8_kernel(const Act8Params p) {
    if constexpr (FLAT) {
        for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < p.n_pieces; i += (long)gridDim.x * 256) {
            if constexpr (READ) read_piece<T, false, GELU>(p, i * VEC, i * VEC, i / kLanesPerRun, VEC);
            else pack_piece<T, false, GELU>(p, i * VEC, i * VEC, i / kLanesPerRun, VEC);
        }
    } else {
        const int sub = threadIdx.x & ((1 << p.lanes_log2) - 1);
        const long step = ((long)gridDim.x * 256) >> p.lanes_log2;
        for (long row = ((long)blockIdx.x * 256 + threadIdx.x) >> p.lanes_log2; row < p.rows; row += step)
            // the lanes of a run stay together: the run's first column decides
            for (int col = sub * VEC; (col & ~(kAct8Group - 1)) < p.E; col += VEC << p.lanes_log2) {
                const long run = row * p.groups + col / kAct8Group;
                if constexpr (READ) read_piece<T, true, GELU>(p, row * p.ldx + col, row * p.E + col, run, p.E - col);
                else pack_piece<T, true, GELU>(p, row * p.ldx + col, row * p.E + col, run, p.E - col);
            }
    }
}

int act8_check(const char *who, int dtype, long M, int E) {
    TC_REQUIRE(dtype == TC_F32 || dtype == TC_BF16, "%s: bad dtype %d", who, dtype);
    TC_REQUIRE(M > 0 && M <= 0x7fffffffL && E > 0 && E <= (1 << 20), "%s: bad shape M=%ld E=%d", who, M, E);
    return TC_OK;
}

Act8Params act8_params(const void *x, long ldx, void *y, void *again, void *codes, void *scales, long M, int E, int esz, bool &flat) {
    Act8Params p{};
    p.x = x; p.ldx = ldx; p.y = y; p.again = again;
    p.codes = static_cast<uint8_t *>(codes);
    p.scales = static_cast<uint8_t *>(scales);
    p.E = E;
    p.groups = (E + kAct8Group - 1) / kAct8Group;
    p.rows = M;
    p.n_pieces = M * (E / VEC);
    p.lanes_log2 = 2;
    while (p.lanes_log2 < 8 && (VEC << p.lanes_log2) < E) ++p.lanes_log2;
    flat = E % kAct8Group == 0 && (!x || (ldx == E && tc_rows_aligned(x, E, esz, VEC))) && tc_rows_aligned(y, E, esz, VEC) &&
           tc_rows_aligned(again, E, esz, VEC) && (uintptr_t)codes % VEC == 0;
    return p;
}

dim3 act8_grid(const Act8Params &p, bool flat) {
    const long lanes = flat ? p.n_pieces : p.rows << p.lanes_log2;
    const long blocks = (lanes + 255) / 256, most = 1L << 20;      // a launch holds fewer than 2^32 threads
    return dim3((unsigned)(blocks < most ? blocks : most));
}

#define TC_A8(T, GELU, READ)                                                                                            \
    do {                                                                                                                \
        if (flat) TC_LAUNCH((act8_kernel<T, true, GELU, READ>), act8_grid(p, true), dim3(256), 0, s, p);                \
        else TC_LAUNCH((act8_kernel<T, false, GELU, READ>), act8_grid(p, false), dim3(256), 0, s, p);                   \
    } while (0)

int pack_call(const char *who, int dtype, const void *x, long ldx, void *act, void *codes, void *scales, long M, int E, bool gelu,
              void *stream) {
    const int rc = act8_check(who, dtype, M, E);
    if (rc != TC_OK) return rc;
    const int esz = dtype == TC_BF16 ? 2 : 4;
    TC_REQUIRE(x && codes && scales && (act || !gelu), "%s: null operand", who);
    TC_REQUIRE(ldx >= E && ((uintptr_t)x | (uintptr_t)act) % esz == 0, "%s: bad row stride or alignment", who);
    hipStream_t s = static_cast<hipStream_t>(stream);
    bool flat;
    const Act8Params p = act8_params(x, ldx, act, nullptr, codes, scales, M, E, esz, flat);
    if (dtype == TC_F32) {
        if (gelu) TC_A8(float, true, false); else TC_A8(float, false, false);
    } else {
        if (gelu) TC_A8(uint16_t, true, false); else TC_A8(uint16_t, false, false);
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
    bool flat;
    const Act8Params p = act8_params(nullptr, 0, out, nullptr, const_cast<void *>(codes), const_cast<void *>(scales), M, E, esz, flat);
    if (dtype == TC_F32) TC_A8(float, false, true);
    else TC_A8(uint16_t, false, true);
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
    bool flat;
    const Act8Params p = act8_params(dy, ld_dy, du, act, const_cast<void *>(codes), const_cast<void *>(scales), M, E, esz, flat);
    if (dtype == TC_F32) TC_A8(float, true, true);
    else TC_A8(uint16_t, true, true);
    TC_CHECK_LAUNCH("tc_dgelu_act8");
    return TC_OK;
}
