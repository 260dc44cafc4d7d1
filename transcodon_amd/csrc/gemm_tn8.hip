// Weight gradient from an 8-bit activation checkpoint (gfx950):
//   dW[N,K] = sum_m dY[m,N] * X[m,K]     dY bf16 [M, ld], X as e4m3 codes [M,K] and one power of two per row and 32 columns
//
// The reduction runs over the rows of both operands, and the scale of X changes with the row: it cannot be taken out of
// the sum.  A code times its power of two is a bf16 number exactly (4 significand bits; from 2^-133 up), so the codes are expanded to
// bf16 on their way into LDS and the product runs on the bf16 matrix cores with f32 accumulators: no rounding but that
// of the f32 sums.  dY goes to LDS by direct loads; fragments of both are taken with the transposing LDS read.
// Two kernels: 128 x 128 output tiles for small products and the last rows, 256 x 256 tiles with two wave groups in
// alternation for large ones.  grid.y splits the rows; the parts are summed in a fixed order, by tc_reduce_slabs or,
// where they are many, by tn8_sum_kernel.
#include "act8.h"
#include <type_traits>

namespace {

constexpr int KT = 64;                         // rows per stage
constexpr int TILE_BYTES = KT * 256;           // 64 rows x 128 bf16
constexpr int STAGE_BYTES = 2 * TILE_BYTES;    // dY + X
constexpr int LDS_BYTES = 2 * STAGE_BYTES;

struct Tn8Params {
    const char *dy;
    const uint8_t *codes, *scales;
    float *out;
    long ld_bytes, slab_elems;
    int M, N, K, groups, nk, splits, tiles_k, accumulate;
};

// 16-byte chunk swizzle of a 256-byte row: the 8 rows that one transposed read touches lie on 8 different 32-byte bank spans
__device__ __forceinline__ int swz(int row) { return ((row & 3) << 2) | (((row >> 2) & 1) << 1); }

// 8 codes of one run as 8 bf16 values
__device__ __forceinline__ u32x4 expand8(uint32_t lo, uint32_t hi, float scale) {
    u32x4 w;
    const uint32_t src[2] = {lo, hi};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)src[k], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)src[k], true);
        w[2 * k] = tc_pack_bf16(a[0] * scale, a[1] * scale);
        w[2 * k + 1] = tc_pack_bf16(b[0] * scale, b[1] * scale);
    }
    return w;
}

__global__ __launch_bounds__(256) void gemm_tn8_kernel(const Tn8Params p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wid >> 1, wj = wid & 1;
    const int tile = tc_xcd_remap(blockIdx.x, gridDim.x);
    const int i0 = (tile / p.tiles_k) * 128, j0 = (tile % p.tiles_k) * 128;
    const int k_begin = (int)((long)p.nk * blockIdx.y / p.splits);
    const int k_end = (int)((long)p.nk * (blockIdx.y + 1) / p.splits);

    // dY: wave w loads rows [16w, 16w+16), 4 rows x 16 chunks of 16 bytes per instruction.  Chunks past the last column read
    // the last one instead (their results are not stored), rows past the last one read the last row.
    const int srow = lane >> 4, schunk = lane & 15;
    long a_col[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = wid * 16 + i * 4 + srow;
        const int col = i0 + ((schunk ^ swz(r)) << 3);
        a_col[i] = 2L * min(col, p.N - 8);
    }
    auto stage_dy = [&](int buf, int kt) {
        char *dst = smem + buf * STAGE_BYTES + wid * 16 * 256;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = min(kt * KT + wid * 16 + i * 4 + srow, p.M - 1);
            __builtin_amdgcn_global_load_lds(TC_GLOBAL_PTR(p.dy + m * p.ld_bytes + a_col[i]), TC_LDS_PTR(dst + i * 1024), 16, 0, 0);
        }
    };
    // X: a thread expands two pieces of 16 codes: rows tid / 8 and tid / 8 + 32, columns 16 (tid % 8) ..
    const int xrow = threadIdx.x >> 3, xpiece = threadIdx.x & 7;
    const int xcol = min(j0 + xpiece * 16, p.K - 16);
    u32x4 xc[2];
    uint32_t xs[2];
    auto load_x = [&](int kt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long m = min(kt * KT + xrow + 32 * i, p.M - 1);
            xc[i] = *reinterpret_cast<const u32x4 *>(p.codes + m * p.K + xcol);
            xs[i] = p.scales[m * p.groups + xcol / kAct8Group];
        }
    };
    auto store_x = [&](int buf) {
        char *dst = smem + buf * STAGE_BYTES + TILE_BYTES;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = xrow + 32 * i;
            const float scale = act8_scale(xs[i]);
            *reinterpret_cast<u32x4 *>(dst + r * 256 + (((2 * xpiece) ^ swz(r)) << 4)) = expand8(xc[i][0], xc[i][1], scale);
            *reinterpret_cast<u32x4 *>(dst + r * 256 + (((2 * xpiece + 1) ^ swz(r)) << 4)) = expand8(xc[i][2], xc[i][3], scale);
        }
    };

    // transposed-read offsets: lane 4q+p of a 16-lane group addresses row q, columns 4p .. 4p+3 of a 4-row x 16-column block and
    // receives the 4 rows of column (lane & 15)
    const int tq = (lane & 15) >> 2, tp = lane & 3, thalf = (lane >> 4) & 1, h2 = lane >> 5;
    int a_off[2][4][2], b_off[2][4][2];        // [block][k-step][lo/hi]
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
                const int row = s * 16 + hi * 8 + 4 * h2 + tq;
                const int ca = wi * 8 + blk * 4 + thalf * 2 + (tp >> 1);
                const int cb = wj * 8 + blk * 4 + thalf * 2 + (tp >> 1);
                a_off[blk][s][hi] = row * 256 + ((ca ^ swz(row)) << 4) + 8 * (tp & 1);
                b_off[blk][s][hi] = TILE_BYTES + row * 256 + ((cb ^ swz(row)) << 4) + 8 * (tp & 1);
            }
    f32x16 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
    auto frag = [&](const char *sb, int lo, int hi) {
        const bf16x4 l = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4 *)(sb + lo));
        const bf16x4 h = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4 *)(sb + hi));
        bf16x8 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) { f[j] = l[j]; f[4 + j] = h[j]; }
        return f;
    };

    if (k_begin < k_end) {
        stage_dy(0, k_begin);
        load_x(k_begin);
        store_x(0);
    }
    for (int kt = k_begin; kt < k_end; ++kt) {
        const int buf = (kt - k_begin) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const bool more = kt + 1 < k_end;
        if (more) {
            stage_dy(buf ^ 1, kt + 1);
            load_x(kt + 1);
        }
        char *sb = smem + buf * STAGE_BYTES;
        const int valid = p.M - kt * KT;           // rows of this stage that exist
        if (valid < KT) {                          // last, partial stage: zero the missing rows of dY
            for (int idx = threadIdx.x; idx < (KT - valid) * 16; idx += 256)
                *reinterpret_cast<u32x4 *>(sb + (valid + (idx >> 4)) * 256 + (idx & 15) * 16) = u32x4{0u, 0u, 0u, 0u};
            __syncthreads();
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            bf16x8 af[2], bf[2];
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                af[blk] = frag(sb, a_off[blk][s][0], a_off[blk][s][1]);
                bf[blk] = frag(sb, b_off[blk][s][0], b_off[blk][s][1]);
            }
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[a], bf[b], acc[a][b], 0, 0, 0);
        }
        if (more) store_x(buf ^ 1);
    }

    float *out = p.out + (long)blockIdx.y * p.slab_elems;
    const int jl = lane & 31;
    auto row_of = [&](int a, int r) { return i0 + wi * 64 + a * 32 + (r & 3) + 8 * (r >> 2) + 4 * h2; };
    auto col_of = [&](int b) { return j0 + wj * 64 + b * 32 + jl; };
    // What is added to is loaded before the first store, all of it under way together (one after the other: 8197 x 2304 x 784 80
    // instead of 65 us); places past the ends read the last one.
    if (p.accumulate) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[a][b][r] += out[(long)min(row_of(a, r), p.N - 1) * p.K + min(col_of(b), p.K - 1)];
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (row_of(a, r) < p.N && col_of(b) < p.K) out[(long)row_of(a, r) * p.K + col_of(b)] = acc[a][b][r];
}

// ------------------------------------------------------------------------------------------
// 256 x 256 output tile, 8 waves in two groups that run half a phase apart: while one wave of a SIMD issues the 16 MFMAs of
// a phase, the other issues that phase's LDS reads, loads and code expansion.  A stage (64 rows) is four half-tiles
// of 64 rows x 256 bytes: A0 A1 = columns i0 .. +127, +128 .. +255 of dY, B0 B1 likewise of X; two stages are in LDS.
// dY comes by LDS-DMA.  X passes through registers: a thread holds 16 codes of each half-tile, loaded one stage before
// they are expanded and two to three stages before they are read, so neither wait stalls.
//   phase 0: read B0, A0    load A1 of stage g+1                                      math quarter (0,0)
//   phase 1: read B1        write B0 of stage g+2, load its codes of stage g+3        math (0,1)
//   phase 2: read A1        load A0 of stage g+2                                      math (1,1)
//   phase 3: -              write B1 of stage g+2, load its codes of stage g+3        math (1,0); stage g+1 complete
// A wave owns 64 (i) x 32 (j) of each quarter of the tile.  Needs whole stages, at least two per split.
// ------------------------------------------------------------------------------------------
namespace big {
constexpr int HALF_BYTES = KT * 256;            // 16 KiB
constexpr int DBUF_BYTES = 4 * HALF_BYTES;
constexpr int SLOT_A0 = 0, SLOT_A1 = HALF_BYTES, SLOT_B0 = 2 * HALF_BYTES, SLOT_B1 = 3 * HALF_BYTES;
constexpr int LDS_BYTES = 2 * DBUF_BYTES;       // 128 KiB
}  // namespace big

// LDS accesses in assembly: the compiler cannot tell them from the LDS-DMA writes in flight and would drain the
// prefetch (vmcnt(0)) in front of each.  Reads are waited for by tn8_wait, through which the fragments are handed on.
template <int OFF>
__device__ __forceinline__ void tn8_read1(unsigned at, bf16x4 &v) {
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(at), "n"(OFF));
}
// two k-steps (32 rows each) of one 16-column block
template <int SLOT>
__device__ __forceinline__ void tn8_read2(unsigned at, bf16x4 (&f)[2][2]) {
    tn8_read1<SLOT>(at, f[0][0]); tn8_read1<SLOT + 4096>(at, f[0][1]);
    tn8_read1<SLOT + 8192>(at, f[1][0]); tn8_read1<SLOT + 8192 + 4096>(at, f[1][1]);
}
__device__ __forceinline__ void tn8_wait(bf16x4 (&f)[2][2], bf16x4 (&g)[2][2]) {
    asm volatile("s_waitcnt lgkmcnt(0)"
                 : "+v"(f[0][0]), "+v"(f[0][1]), "+v"(f[1][0]), "+v"(f[1][1]), "+v"(g[0][0]), "+v"(g[0][1]), "+v"(g[1][0]),
                   "+v"(g[1][1]));
}
__device__ __forceinline__ bf16x8 tn8_join(bf16x4 l, bf16x4 h) { return __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7); }
template <int OFF>
__device__ __forceinline__ void tn8_write(unsigned at, u32x4 v) {
    asm volatile("ds_write_b128 %0, %1 offset:%2" : : "v"(at), "v"(v), "n"(OFF) : "memory");
}
// 8 codes of one run as 8 bf16 values, scaled by the conversion itself
__device__ __forceinline__ u32x4 tn8_expand(uint32_t lo, uint32_t hi, float scale) {
    u32x4 w;
    w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return w;
}

#define TN8_XBAR()                                 \
    do {                                           \
        __builtin_amdgcn_sched_barrier(0);         \
        __builtin_amdgcn_s_barrier();              \
        __builtin_amdgcn_sched_barrier(0);         \
    } while (0)

__global__ __launch_bounds__(512) void gemm_tn8_256_kernel(const Tn8Params p) {
    using namespace big;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wid >> 2, wc = wid & 3;
    const int i0 = (blockIdx.x / p.tiles_k) * 256, j0 = (blockIdx.x % p.tiles_k) * 256;
    const int k_begin = (int)((long)p.nk * blockIdx.y / p.splits);
    const int nkt = (int)((long)p.nk * (blockIdx.y + 1) / p.splits) - k_begin;      // >= 2 (host)

    // dY: a half-tile is 16 pieces of 4 rows x 256 bytes, this wave moves pieces 2 wid, 2 wid + 1.  Columns past the last one
    // read the last 16 bytes instead (their results are not stored).  Offsets are from the split's first row (host: < 4 GiB).
    const int srow = lane >> 4, schunk = lane & 15;
    unsigned a_src[2][2];                        // [half][piece]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = (wid * 2 + i) * 4 + srow;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            a_src[h][i] = (unsigned)(r * p.ld_bytes) + 2u * (unsigned)min(i0 + h * 128 + ((schunk ^ swz(r)) << 3), p.N - 8);
    }
    const long row0 = (long)k_begin * KT;
    const __amdgpu_buffer_rsrc_t rsrc_a = tc_buffer_rsrc(p.dy + row0 * p.ld_bytes);
    auto stage_a = [&](int slot_off, const unsigned (&src)[2], int kt) {
        char *dst = smem + slot_off + wid * 2048;
        const unsigned off = (unsigned)((long)kt * KT * p.ld_bytes);
        tc_blds16(rsrc_a, src[0], off, dst);
        tc_blds16(rsrc_a, src[1], off, dst + 1024);
    };
    // X: row tid / 8 of the stage, codes 16 (tid % 8) .. of both half-tiles
    const int xrow = threadIdx.x >> 3, xpiece = threadIdx.x & 7;
    const __amdgpu_buffer_rsrc_t rsrc_c = tc_buffer_rsrc(p.codes + row0 * p.K), rsrc_s = tc_buffer_rsrc(p.scales + row0 * p.groups);
    unsigned c_src[2], s_src[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int col = min(j0 + h * 128 + xpiece * 16, p.K - 16);
        c_src[h] = (unsigned)(xrow * p.K + col);
        s_src[h] = (unsigned)(xrow * p.groups + col / kAct8Group);
    }
    u32x4 xc[2];
    uint32_t xs[2];
    auto load_x = [&](auto h_c, int kt) {
        constexpr int h = decltype(h_c)::value;
        xc[h] = __builtin_amdgcn_raw_buffer_load_b128(rsrc_c, (int)c_src[h], (int)((unsigned)kt * KT * (unsigned)p.K), 0);
        xs[h] = __builtin_amdgcn_raw_buffer_load_b8(rsrc_s, (int)s_src[h], (int)((unsigned)kt * KT * (unsigned)p.groups), 0);
    };
    const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) char *)smem;
    const unsigned x_at = lds0 + xrow * 256 + (((2 * xpiece) ^ swz(xrow)) << 4);     // the other 16 bytes: chunk ^ 1
    auto write_x = [&](auto h_c, int buf_off) {
        constexpr int h = decltype(h_c)::value;
        const float scale = act8_scale(xs[h]);
        tn8_write<(h ? SLOT_B1 : SLOT_B0)>(x_at + buf_off, tn8_expand(xc[h][0], xc[h][1], scale));
        tn8_write<(h ? SLOT_B1 : SLOT_B0)>((x_at ^ 16) + buf_off, tn8_expand(xc[h][2], xc[h][3], scale));
    };

    // Transposed-read offsets inside a half-tile (row pitch 256 B): 16-lane group tg addresses rows 4 tg + tq, bytes 8 tp .. of a
    // 16-column block and receives the 4 rows of column lane & 15; a fragment of the 16x16x32 MFMA is that read and the one
    // 16 rows further, in the same order for both operands.
    const int tg = lane >> 4, tq = (lane & 15) >> 2, tp = lane & 3, c16 = lane & 15;
    const int row_l = 4 * tg + tq, sw = swz(row_l);
    unsigned a_addr[4], b_addr[2];
#pragma unroll
    for (int blk = 0; blk < 4; ++blk)
        a_addr[blk] = lds0 + row_l * 256 + (((wr * 8 + blk * 2 + (tp >> 1)) ^ sw) << 4) + 8 * (tp & 1);
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
        b_addr[blk] = lds0 + row_l * 256 + (((wc * 4 + blk * 2 + (tp >> 1)) ^ sw) << 4) + 8 * (tp & 1);

    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    // ---- prologue: stages 0 and 1 but A1 of stage 1; codes of stage 2 ----
    // The last loads are in the order of the loop's phases 1 to 3, so that the counted waits the compiler places are the
    // same on the way in and around.  For the same reason the loop has no branch: past the last stage it loads the last one
    // again, into places that nobody reads.
    stage_a(SLOT_A0, a_src[0], 0);
    stage_a(SLOT_A1, a_src[1], 0);
    load_x(I0{}, 0);
    load_x(I1{}, 0);
    write_x(I0{}, 0);
    write_x(I1{}, 0);
    load_x(I0{}, 1);
    load_x(I1{}, 1);
    write_x(I0{}, DBUF_BYTES);
    write_x(I1{}, DBUF_BYTES);
    const int ahead = min(2, nkt - 1);
    load_x(I0{}, ahead);
    __builtin_amdgcn_sched_barrier(0);
    stage_a(DBUF_BYTES + SLOT_A0, a_src[0], 1);
    __builtin_amdgcn_sched_barrier(0);
    load_x(I1{}, ahead);
    asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
    TN8_XBAR();
    if (wr == 1) TN8_XBAR();                      // group 1 runs half a phase behind

    f32x4 acc[8][4];                              // [mq * 4 + i block][nq * 2 + j block], D[i][j]
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int g = 0; g < nkt; ++g) {
        const int cur = (g & 1) * DBUF_BYTES, nxt = DBUF_BYTES - cur;
        bf16x4 bq[2][2][2][2];                    // [nq][j block][k-step][lower / upper 16 rows]
        bf16x4 af[4][2][2];                       // [i block][k-step][lower / upper] of the current mq
        auto read_b = [&](auto nq_c) {
            constexpr int nq = decltype(nq_c)::value;
            tn8_read2<(nq ? SLOT_B1 : SLOT_B0)>(b_addr[0] + cur, bq[nq][0]);
            tn8_read2<(nq ? SLOT_B1 : SLOT_B0)>(b_addr[1] + cur, bq[nq][1]);
        };
        auto read_a = [&](auto mq_c, auto half_c) {          // i blocks 2 half, 2 half + 1
            constexpr int mq = decltype(mq_c)::value, hf = decltype(half_c)::value;
            tn8_read2<(mq ? SLOT_A1 : SLOT_A0)>(a_addr[2 * hf] + cur, af[2 * hf]);
            tn8_read2<(mq ? SLOT_A1 : SLOT_A0)>(a_addr[2 * hf + 1] + cur, af[2 * hf + 1]);
        };
        auto math = [&](int mq, int nq) {
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                    for (int ib = 0; ib < 4; ++ib)
                        acc[mq * 4 + ib][nq * 2 + jb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            tn8_join(af[ib][s][0], af[ib][s][1]), tn8_join(bq[nq][jb][s][0], bq[nq][jb][s][1]),
                            acc[mq * 4 + ib][nq * 2 + jb], 0, 0, 0);
            __builtin_amdgcn_s_setprio(0);
        };
        const int far = min(g + 3, nkt - 1);
        // ---- phase 0 ----
        stage_a(nxt + SLOT_A1, a_src[1], min(g + 1, nkt - 1));
        read_b(I0{});
        read_a(I0{}, I0{});
        // the B0 reads (8 of the 16 issued; the counter holds 15): their slot is written in phase 1
        asm volatile("s_waitcnt lgkmcnt(8)" ::: "memory");
        read_a(I0{}, I1{});
        TN8_XBAR();
        tn8_wait(bq[0][0], bq[0][1]); tn8_wait(af[0], af[1]); tn8_wait(af[2], af[3]);
        math(0, 0);
        TN8_XBAR();
        // ---- phase 1 ----
        write_x(I0{}, cur);
        load_x(I0{}, far);
        read_b(I1{});
        TN8_XBAR();
        tn8_wait(bq[1][0], bq[1][1]);
        math(0, 1);
        TN8_XBAR();
        // ---- phase 2 ----
        stage_a(cur + SLOT_A0, a_src[0], min(g + 2, nkt - 1));
        read_a(I1{}, I0{});
        read_a(I1{}, I1{});
        TN8_XBAR();
        tn8_wait(af[0], af[1]); tn8_wait(af[2], af[3]);
        math(1, 1);
        TN8_XBAR();
        // ---- phase 3 ----
        write_x(I1{}, cur);
        load_x(I1{}, far);
        // all but the loads of phases 1 to 3: A1 of stage g+1 has landed, and this wave's LDS writes
        asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
        TN8_XBAR();
        math(1, 0);
        TN8_XBAR();
    }
    if (wr == 0) TN8_XBAR();                      // pairs with group 1's last barrier
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // no LDS-DMA write may outlive the workgroup

    float *out = p.out + (long)blockIdx.y * p.slab_elems;
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int j = j0 + (b >> 1) * 128 + wc * 32 + (b & 1) * 16 + c16;
            const int i = i0 + (a >> 2) * 128 + wr * 64 + (a & 3) * 16 + 4 * tg;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (i + r < p.N && j < p.K) {
                    float *to = out + (long)(i + r) * p.K + j;
                    *to = p.accumulate ? *to + acc[a][b][r] : acc[a][b][r];
                }
        }
}

// Sum of many parts of a small gradient: 64 columns of four values a workgroup, 16 waves that take every 16th part each and
// are added in order.  (tc_reduce_slabs gives a thread all parts of its values, one load after the other.)
__global__ __launch_bounds__(1024) void tn8_sum_kernel(const float *__restrict__ slabs, float *__restrict__ out, int S, long n4, int accumulate) {
    __shared__ f32x4 red[16][64];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const long i = (long)blockIdx.x * 64 + c;
    f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
    if (i < n4)
#pragma unroll 8
        for (int k = r; k < S; k += 16) sum += *reinterpret_cast<const f32x4 *>(slabs + 4 * (k * n4 + i));
    red[r][c] = sum;
    __syncthreads();
    if (r == 0 && i < n4) {
        for (int k = 1; k < 16; ++k) sum += red[k][c];
        if (accumulate) sum += *reinterpret_cast<const f32x4 *>(out + 4 * i);
        *reinterpret_cast<f32x4 *>(out + 4 * i) = sum;
    }
}

bool tn8_dims_ok(long M, int N, int K) {
    return M > 0 && M <= 0x7fffffffL - KT && N > 0 && K > 0 && N % 8 == 0 && K % 16 == 0 && N <= (1 << 20) && K <= (1 << 20) &&
           (long)((N + 127) / 128) * ((K + 127) / 128) <= (1 << 22);
}

struct Tn8Plan {
    bool big;                // 256 x 256 tiles over the whole stages, the rows behind them by the small kernel
    int splits;              // row splits, and parts of the sum
};
constexpr int kManySlabs = 16;
// What the parts of a sum may take: this, or a quarter of the operands' bytes.  More of them gain little where products are that
// large (231953 x 13736 x 12176: 7 parts, 4.7 GB, 65.7 ms; 3 parts, 2.0 GB, 66.9 ms; 20003 x 16384 x 4096: 2 parts 2.35 ms, 1 part 2.25).
constexpr long kPartBytes = 128L << 20;
// Which kernel and how many row splits: the least estimated time over both kernels and up to 256 splits, in nanoseconds.
// A stage takes a large tile 1.9 us on a full chip (220 us at 65536 x 2304 x 768: 114 stages), a small one 1 us while
// there is one workgroup per CU and 0.6 us more for each further one (kernel trace, 768 x 768 on 36 CUs: 5.8 us for 64 rows, 0.8 us
// for each further 64; the 2 us taken here for start and end are 5, but for every number of splits alike); a part of the sum costs its slab written and read at
// 6.5 TB/s, and more than one the summing launch.
Tn8Plan tn8_plan(long M, long ld_dy, int N, int K) {
    Tn8Plan best{};
    long least = -1;
    const long nk = (M + KT - 1) / KT, whole = M / KT;
    const long large = (long)((N + 255) / 256) * ((K + 255) / 256), small = (long)((N + 127) / 128) * ((K + 127) / 128);
    const long quarter = M * (2L * N + K) / 4, most = quarter > kPartBytes ? quarter : kPartBytes;
    auto parts = [&](long slabs) { return slabs > 1 ? 4000 + slabs * N * K * 8 / 6500 : 0; };
    for (long s = 1; s <= 256; s += s < 16 ? 1 : s < 64 ? 4 : 16) {
        if (s > 1 && s * N * K * 4 > most) break;
        if (s >= kManySlabs && (long)N * K > (1L << 29)) break;      // tn8_sum_kernel's launch holds fewer than 2^32 threads
        if (s <= nk) {
            const long wgs = small * s;
            const long ns = 2000 + (nk + s - 1) / s * (400 + 600 * (wgs > 256 ? wgs : 256) / 256) + parts(s);
            if (least < 0 || ns < least) {
                least = ns;
                best = Tn8Plan{false, (int)s};
            }
        }
        // offsets inside a split, with the stages loaded ahead, are 32 bits
        const long rows = (whole / s + 4) * KT;
        if (whole >= 2 * s && rows * ld_dy * 2 < (1L << 32) && rows * K < (1L << 32)) {
            const int rest = M % KT != 0;          // the rows behind the whole stages: one more launch
            const long ns = 3000 + (whole + s - 1) / s * 1900 * ((large * s + 255) / 256) + 5000 * rest + parts(s);
            if (ns < least) {
                least = ns;
                best = Tn8Plan{true, (int)s};
            }
        }
    }
    return best;
}

}  // namespace

extern "C" size_t tc_gemm_tn_act8_workspace_bytes(long M, long ld_dy, int N, int K) {
    if (!tn8_dims_ok(M, N, K) || ld_dy < N) return 0;
    const int parts = tn8_plan(M, ld_dy, N, K).splits;
    return parts > 1 ? (size_t)parts * N * K * sizeof(float) : 16;
}

extern "C" int tc_gemm_tn_act8(const void *dy, long ld_dy, const void *codes, const void *scales, float *dW, long M, int N, int K,
                               int accumulate, void *workspace, size_t workspace_bytes, void *stream) {
    TC_REQUIRE(dy && codes && scales && dW && workspace, "tc_gemm_tn_act8: null operand");
    TC_REQUIRE(tn8_dims_ok(M, N, K), "tc_gemm_tn_act8: M=%ld N=%d K=%d (N a multiple of 8, K of 16)", M, N, K);
    TC_REQUIRE(ld_dy >= N && ld_dy % 8 == 0, "tc_gemm_tn_act8: row stride %ld of dY (at least N, a multiple of 8)", ld_dy);
    TC_REQUIRE(tc_aligned16(dy) && tc_aligned16(codes) && tc_aligned16(dW) && tc_aligned16(workspace),
               "tc_gemm_tn_act8: operands must be 16-byte aligned");
    const size_t need = tc_gemm_tn_act8_workspace_bytes(M, ld_dy, N, K);
    if (workspace_bytes < need) {
        tc_set_error("tc_gemm_tn_act8: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return TC_ENOSPC;
    }
    const Tn8Plan w = tn8_plan(M, ld_dy, N, K);
    Tn8Params p{};
    p.dy = static_cast<const char *>(dy);
    p.codes = static_cast<const uint8_t *>(codes);
    p.scales = static_cast<const uint8_t *>(scales);
    p.ld_bytes = ld_dy * 2;
    p.M = (int)M; p.N = N; p.K = K;
    p.groups = (K + kAct8Group - 1) / kAct8Group;
    p.splits = w.splits;
    p.out = w.splits > 1 ? static_cast<float *>(workspace) : dW;
    p.slab_elems = (long)N * K;
    p.accumulate = w.splits > 1 ? 0 : accumulate;
    hipStream_t s = static_cast<hipStream_t>(stream);
    static_assert(LDS_BYTES <= 64 * 1024, "no attribute needed");
    const dim3 small_grid((unsigned)(((N + 127) / 128) * ((K + 127) / 128)), (unsigned)w.splits);
    TcProfScope prof(TC_PROF_GEMM, s, 2.0 * (double)M * N * K);
    if (w.big) {
        // per device; setting it again is harmless, so threads need no lock
        static bool attr_set[64];
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        if (e == hipSuccess && (dev >= 64 || !attr_set[dev])) {
            e = hipFuncSetAttribute(reinterpret_cast<const void *>(gemm_tn8_256_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    big::LDS_BYTES);
            if (e == hipSuccess && dev < 64) attr_set[dev] = true;
        }
        if (e != hipSuccess) {
            tc_set_error("tc_gemm_tn_act8: hipFuncSetAttribute: %s", hipGetErrorString(e));
            return TC_ELAUNCH;
        }
        p.nk = (int)(M / KT);
        p.tiles_k = (K + 255) / 256;
        TC_LAUNCH(gemm_tn8_256_kernel, dim3((unsigned)(((N + 255) / 256) * p.tiles_k), (unsigned)w.splits), dim3(512), big::LDS_BYTES, s, p);
        if (M % KT != 0) {                         // the last rows: added to the first part
            const long done = M / KT * KT;
            Tn8Params t = p;
            t.accumulate = 1;
            t.dy += done * p.ld_bytes;
            t.codes += done * K;
            t.scales += done * p.groups;
            t.M = (int)(M - done);
            t.nk = t.splits = 1;
            t.tiles_k = (K + 127) / 128;
            TC_LAUNCH(gemm_tn8_kernel, dim3(small_grid.x, 1), dim3(256), LDS_BYTES, s, t);
        }
    } else {
        p.nk = (int)((M + KT - 1) / KT);
        p.tiles_k = (K + 127) / 128;
        TC_LAUNCH(gemm_tn8_kernel, small_grid, dim3(256), LDS_BYTES, s, p);
    }
    if (w.splits > kManySlabs) {
        const long n4 = (long)N * K / 4;
        TC_LAUNCH(tn8_sum_kernel, dim3((unsigned)((n4 + 63) / 64)), dim3(1024), 0, s, p.out, dW, w.splits, n4, accumulate);
    }
    TC_CHECK_LAUNCH("tc_gemm_tn_act8");
    return w.splits > 1 && w.splits <= kManySlabs ? tc_reduce_slabs(p.out, dW, w.splits, (long)N * K, accumulate, stream) : TC_OK;
}
