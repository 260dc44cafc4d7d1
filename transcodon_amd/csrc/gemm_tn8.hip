// Weight gradient from an 8-bit activation checkpoint (gfx950):
//   dW[N,K] = sum_m dY[m,N] * X[m,K]     dY bf16 [M, ld], X as e4m3 codes [M,K] and one power of two per row and 32 columns
//
// The reduction runs over the rows of both operands, and the scale of X changes with the row: it cannot be taken out of
// the sum.  A code times its power of two is a bf16 number exactly (4 significand bits), so the codes are expanded to
// bf16 on their way into LDS and the product runs on the bf16 matrix cores with f32 accumulators: no rounding but that
// of the f32 sums.  dY goes to LDS by direct loads; fragments of both are taken with the transposing LDS read.
// Workgroup: 256 threads, 128 x 128 output tile, 2 x 2 waves of 64 x 64.  grid.y splits the rows; the parts are summed
// by tc_reduce_slabs in a fixed order.
#include "act8.h"

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
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int j = j0 + wj * 64 + b * 32 + jl;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = i0 + wi * 64 + a * 32 + (r & 3) + 8 * (r >> 2) + 4 * h2;
                if (i < p.N && j < p.K) {
                    float *to = out + (long)i * p.K + j;
                    *to = p.accumulate ? *to + acc[a][b][r] : acc[a][b][r];
                }
            }
        }
}

bool tn8_dims_ok(long M, int N, int K) {
    return M > 0 && M <= 0x7fffffffL - KT && N > 0 && K > 0 && N % 8 == 0 && K % 16 == 0 && N <= (1 << 20) && K <= (1 << 20) &&
           (long)((N + 127) / 128) * ((K + 127) / 128) <= (1 << 22);
}

// Row splits: about four workgroups per CU, no more than there are stages
int tn8_splits(long M, int N, int K) {
    const long tiles = (long)((N + 127) / 128) * ((K + 127) / 128), nk = (M + KT - 1) / KT;
    long s = 1024 / tiles;
    s = s < 1 ? 1 : s > 64 ? 64 : s;
    return (int)(s < nk ? s : nk);
}

}  // namespace

extern "C" size_t tc_gemm_tn_act8_workspace_bytes(long M, int N, int K) {
    if (!tn8_dims_ok(M, N, K)) return 0;
    const int splits = tn8_splits(M, N, K);
    return splits > 1 ? (size_t)splits * N * K * sizeof(float) : 16;
}

extern "C" int tc_gemm_tn_act8(const void *dy, long ld_dy, const void *codes, const void *scales, float *dW, long M, int N, int K,
                               int accumulate, void *workspace, size_t workspace_bytes, void *stream) {
    TC_REQUIRE(dy && codes && scales && dW && workspace, "tc_gemm_tn_act8: null operand");
    TC_REQUIRE(tn8_dims_ok(M, N, K), "tc_gemm_tn_act8: M=%ld N=%d K=%d (N a multiple of 8, K of 16)", M, N, K);
    TC_REQUIRE(ld_dy >= N && ld_dy % 8 == 0, "tc_gemm_tn_act8: row stride %ld of dY (at least N, a multiple of 8)", ld_dy);
    TC_REQUIRE(tc_aligned16(dy) && tc_aligned16(codes) && tc_aligned16(dW) && tc_aligned16(workspace),
               "tc_gemm_tn_act8: operands must be 16-byte aligned");
    const size_t need = tc_gemm_tn_act8_workspace_bytes(M, N, K);
    if (workspace_bytes < need) {
        tc_set_error("tc_gemm_tn_act8: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return TC_ENOSPC;
    }
    Tn8Params p{};
    p.dy = static_cast<const char *>(dy);
    p.codes = static_cast<const uint8_t *>(codes);
    p.scales = static_cast<const uint8_t *>(scales);
    p.ld_bytes = ld_dy * 2;
    p.M = (int)M; p.N = N; p.K = K;
    p.groups = (K + kAct8Group - 1) / kAct8Group;
    p.nk = (int)((M + KT - 1) / KT);
    p.splits = tn8_splits(M, N, K);
    p.tiles_k = (K + 127) / 128;
    p.out = p.splits > 1 ? static_cast<float *>(workspace) : dW;
    p.slab_elems = (long)N * K;
    p.accumulate = p.splits > 1 ? 0 : accumulate;
    hipStream_t s = static_cast<hipStream_t>(stream);
    static_assert(LDS_BYTES <= 64 * 1024, "no attribute needed");
    {
        TcProfScope prof(TC_PROF_GEMM, s, 2.0 * (double)M * N * K);
        TC_LAUNCH(gemm_tn8_kernel, dim3((unsigned)(((N + 127) / 128) * p.tiles_k), (unsigned)p.splits), dim3(256), LDS_BYTES, s, p);
    }
    TC_CHECK_LAUNCH("tc_gemm_tn_act8");
    return p.splits > 1 ? tc_reduce_slabs(p.out, dW, p.splits, (long)N * K, accumulate, stream) : TC_OK;
}
