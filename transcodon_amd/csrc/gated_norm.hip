// The end of one residual block and the start of the next in one pass:
//
//   n     = norm_post(y) * g1 + b1                norm after the block (y: the block's output)
//   x_out = res_scale * x + gate o n              gate: a row of [G,E] for M / G consecutive rows, or none
//   h     = norm_pre(x_out) * g2 + b2             norm before the next block (left out where g2 is null)
//
// and its backward pass.  norm(t) = (t - mean) * rstd, or t * rstd for root-mean-square norms (mean = 0).  The residual
// stream and all arithmetic are f32; y, h and their gradients are f32 or bf16.
//
// A team of W waves owns a row at a time and keeps it in registers, so every operand is read from memory once; deviations are
// summed after the mean is known.  HBM bound: 65536 x 768 in bf16 with 64 gate rows 109 us forward (604 MB, 5.5 TB/s; a
// large copy: 4.9) and 188 us backward (907 MB, 4.8 TB/s).  The backward pass gives each team a run of
// neighbouring rows and keeps the column sums (gradients of the norms' vectors and of the gate) in registers; teams of
// a workgroup are added in LDS, workgroups by a second kernel, always in the same order.
#include "row_io.h"

namespace {

constexpr int VEC = 4;                       // neighbouring values of a row that a lane loads at a time

template <int W>
struct Team {                                // W waves that work on one row
    float (*lds)[2][W];                      // [turn][value][wave]
    int wave, turn = 0;
    // sums of a and b over the team's lanes, on every lane
    __device__ __forceinline__ void sum2(float &a, float &b) {
        a = tc_wave_sum(a);
        b = tc_wave_sum(b);
        if constexpr (W > 1) {
            // two buffers in turn: a wave writes one only after the barrier that follows every read of it
            if ((threadIdx.x & 63) == 0) { lds[turn][0][wave] = a; lds[turn][1][wave] = b; }
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) { a += lds[turn][0][w]; b += lds[turn][1][w]; }
            turn ^= 1;
        }
    }
    __device__ __forceinline__ float sum(float a) {
        float unused = 0.f;
        sum2(a, unused);
        return a;
    }
};

// The columns of a lane, NC pieces of VEC.  Every piece has VEC columns of the row: one that would pass its end is moved back, to
// columns that other lanes have as well.  Those come to the same values, so they may be stored twice, but a sum counts a piece's
// columns from `skip` on only.  So loads and stores stand in no branch: where paths with different numbers of them meet, the
// compiler waits for all that are under way (8192 x 4098 bf16 forward: 160 us with the row's end in a branch of its own, 92 so).
template <bool LOOSE, int W, int NC, int VEC>
struct Pieces {
    int col[NC], skip[NC];
    __device__ __forceinline__ Pieces(int wave, int E) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int want = ((wave + c * W) * 64 + (int)(threadIdx.x & 63)) * VEC;
            col[c] = min(want, E - VEC);
            skip[c] = want - col[c];
        }
    }
    __device__ __forceinline__ bool counts(int c, int j) const { return LOOSE ? j >= skip[c] : skip[c] == 0; }
};

// mean and 1 / sqrt(variance + eps) of a row held as v[NC][VEC]
template <bool LOOSE, int W, int NC, int VEC>
__device__ __forceinline__ void row_stats(Team<W> &team, const Pieces<LOOSE, W, NC, VEC> &at, const float (&v)[NC][VEC], int E, int rms,
                                          float eps, float &mean, float &rstd) {
    mean = 0.f;
    if (!rms) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += at.counts(c, j) ? v[c][j] : 0.f;
        mean = team.sum(s) / (float)E;
    }
    float q = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float d = at.counts(c, j) ? v[c][j] - mean : 0.f;
            q += d * d;
        }
    rstd = rsqrtf(team.sum(q) / (float)E + eps);
}

// Has the loads that v came from arrive here.
template <int NC, int VEC>
__device__ __forceinline__ void arrived(float (&v)[NC][VEC]) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) asm volatile("" : "+v"(v[c][j]));
}

struct NormParams {
    const void *y, *gate;
    const float *x, *g1, *b1, *g2, *b2;
    float *x_out, *stats;
    void *h;
    // backward
    const void *dh;
    const float *dx_out;
    void *dy;
    float *dx, *d_gate, *ws;
    float *d_vec[4];                         // gradients of g1, b1, g2, b2 (null: not wanted)
    int accumulate;                          // bit v: add to d_vec[v]; bit 4: add to d_gate
    long ldy, ldx, ld_dh, ld_dxo;
    int M, E, rms;
    int rows_per_gate;                       // M / G (M without a gate)
    float res_scale, eps1, eps2;
    // backward: team t owns rows [t * rows_per_team, ...) of whole gate groups, or a part of one group
    int teams, rows_per_team, teams_per_group;
};

template <typename T, typename TG, bool LOOSE, int W, int NC, int VEC>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void gated_norm_kernel(const NormParams p) {
    __shared__ float red[2][2][W];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Team<W> team{red, W == 1 ? 0 : wave};
    constexpr int kTeams = W == 1 ? 4 : 1;
    const Pieces<LOOSE, W, NC, VEC> at(W == 1 ? 0 : wave, p.E);
    // One or two teams of many waves fill a CU and meet at barriers: they ask for their next row before they work on this one and
    // keep the vectors, which are more bytes than a row (8192 x 8192 bf16: 183 -> 157 us, 4096 wide 96 -> 79).  Smaller teams
    // find others to hide their loads behind.
    constexpr bool kAhead = W > 4;
    struct Vectors {
        float g1[NC][VEC], b1[NC][VEC], gate[NC][VEC], g2[NC][VEC], b2[NC][VEC];
    } k;
    auto load_vectors = [&]() {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) k.b1[c][j] = k.g2[c][j] = k.b2[c][j] = 0.f;
            tc_load_row<float, VEC, LOOSE>(p.g1 + at.col[c], k.g1[c]);
            if (p.b1) tc_load_row<float, VEC, LOOSE>(p.b1 + at.col[c], k.b1[c]);
            if (p.g2) tc_load_row<float, VEC, LOOSE>(p.g2 + at.col[c], k.g2[c]);
            if (p.b2) tc_load_row<float, VEC, LOOSE>(p.b2 + at.col[c], k.b2[c]);
        }
    };
    auto load_gate = [&](long row) {
        const long gate_row = (long)((unsigned)row / (unsigned)p.rows_per_gate) * p.E;      // rows are below 2^31
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) k.gate[c][j] = 1.f;
            if (p.gate) tc_load_row<TG, VEC, LOOSE>(static_cast<const TG *>(p.gate) + gate_row + at.col[c], k.gate[c]);
        }
    };
    struct Row {
        typename TcRaw<T, VEC>::type y[NC];
        typename TcRaw<float, VEC>::type x[NC];
    } next;
    auto request = [&](long row) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            next.y[c] = tc_raw_load<T, VEC, LOOSE>(static_cast<const T *>(p.y) + row * p.ldy + at.col[c]);
            next.x[c] = tc_raw_load<float, VEC, LOOSE>(p.x + row * p.ldx + at.col[c]);
        }
    };
    const long step = (long)gridDim.x * kTeams;
    long row = (long)blockIdx.x * kTeams + (W == 1 ? wave : 0);
    if (kAhead && row < p.M) {
        load_vectors();
        request(row);
        arrived(k.g1); arrived(k.b1); arrived(k.g2); arrived(k.b2);
#pragma unroll
        for (int c = 0; c < NC; ++c) asm volatile("" : "+v"(next.y[c]), "+v"(next.x[c]));
    }
    for (; row < p.M; row += step) {
        if (!kAhead) request(row);
        float yv[NC][VEC], xv[NC][VEC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            tc_raw_widen<T, VEC>(next.y[c], yv[c]);
            tc_raw_widen<float, VEC>(next.x[c], xv[c]);
        }
        if (!kAhead) load_vectors();
        load_gate(row);
        if (kAhead) request(row + step < p.M ? row + step : row);
        if (W > 1) arrived(xv);                  // x_out may be x: before the team's next barrier, which is before its stores
        float mean1, rstd1;
        row_stats(team, at, yv, p.E, p.rms, p.eps1, mean1, rstd1);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                xv[c][j] = p.res_scale * xv[c][j] + ((yv[c][j] - mean1) * rstd1 * k.g1[c][j] + k.b1[c][j]) * k.gate[c][j];
            tc_store_row<float, VEC, LOOSE>(p.x_out + row * p.E + at.col[c], xv[c]);
        }
        float mean2 = 0.f, rstd2 = 0.f;
        if (p.g2) {
            row_stats(team, at, xv, p.E, p.rms, p.eps2, mean2, rstd2);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) xv[c][j] = (xv[c][j] - mean2) * rstd2 * k.g2[c][j] + k.b2[c][j];
                tc_store_row<T, VEC, LOOSE>(static_cast<T *>(p.h) + row * p.E + at.col[c], xv[c]);
            }
        }
        if (p.stats && (W == 1 ? threadIdx.x & 63 : threadIdx.x) == 0) *reinterpret_cast<f32x4 *>(p.stats + row * 4) = f32x4{mean1, rstd1, mean2, rstd2};
    }
}

// Gradient.  With D = d(loss)/d(x_out) in full:
//   x^ = (x_out - mean2) rstd2    D = dx_out + rstd2 (p - mean(p) - x^ mean(p x^)),  p = dh o g2
//   y^ = (y - mean1) rstd1        dn = D o gate     dy = rstd1 (q - mean(q) - y^ mean(q y^)),  q = dn o g1
//   dx = res_scale D    d_gate = sum D o n    d_g1 = sum dn o y^   d_b1 = sum dn   d_g2 = sum dh o x^   d_b2 = sum dh
// (root-mean-square norms: without the mean(p), mean(q) terms).
template <typename T, typename TG, bool LOOSE, int W, int NC, int VEC>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void gated_norm_bwd_kernel(const NormParams p) {
    extern __shared__ float sums[];          // [team][E] (W == 1)
    __shared__ float red[2][2][W];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Team<W> team{red, W == 1 ? 0 : wave};
    constexpr int kTeams = W == 1 ? 4 : 1;   // teams of a workgroup
    const int t = blockIdx.x * kTeams + (W == 1 ? wave : 0);
    const Pieces<LOOSE, W, NC, VEC> at(W == 1 ? 0 : wave, p.E);
    float acc[4][NC][VEC], dgt[NC][VEC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            acc[0][c][j] = acc[1][c][j] = acc[2][c][j] = acc[3][c][j] = 0.f;
            dgt[c][j] = 0.f;
        }
    // rows of this team
    long begin, end;
    if (p.teams_per_group > 0) {
        const int g = t / p.teams_per_group, part = t - g * p.teams_per_group;
        begin = (long)g * p.rows_per_gate + (long)part * p.rows_per_team;
        end = min((long)(g + 1) * p.rows_per_gate, begin + p.rows_per_team);
    } else {
        begin = (long)t * p.rows_per_team;
        end = min((long)p.M, begin + p.rows_per_team);
    }
    if (t >= p.teams) begin = end = 0;
    const float inv_e = 1.0f / (float)p.E;
    // A row's operands as they were loaded.  The next row is requested before this one is worked on, since three dependent
    // row reductions leave a wave idle otherwise, and the vectors stay in registers, the gate's row until its group ends
    // (loading them again for every row: 65536 x 768 bf16 208 instead of 194 us).  More than eight waves leave too few registers
    // for either.
    // No load or store of the loop stands in a branch but those of a new gate row: an operand that is not there is read from one
    // row of another, and what is loaded before the loop is waited for there.
    constexpr bool kAhead = W <= 8, kKeep = W <= 8;
    const T *const dh_rows = p.g2 ? static_cast<const T *>(p.dh) : static_cast<const T *>(p.y);
    const float *const d_rows = p.dx_out ? p.dx_out : p.x;
    const long ldx = p.g2 ? p.ldx : 0, ld_dh = p.g2 ? p.ld_dh : 0, ld_d = p.dx_out ? p.ld_dxo : 0;
    struct Row {
        typename TcRaw<T, VEC>::type y[NC], dh[NC];
        typename TcRaw<float, VEC>::type x[NC], d[NC];
        typename TcRaw<TG, VEC>::type gate[NC];
        f32x4 st;
    } next;
    auto gate_row_of = [&](long row) { return (long)((unsigned)row / (unsigned)p.rows_per_gate) * p.E; };      // rows are below 2^31
    long kept_gate = -1;                     // the row of the gate that `next` or kgt holds
    bool fresh_gate = false;
    auto request = [&](long row) {
        if (kKeep && p.gate) {
            fresh_gate = gate_row_of(row) != kept_gate;
            if (fresh_gate) {
                kept_gate = gate_row_of(row);
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    next.gate[c] = tc_raw_load<TG, VEC, LOOSE>(static_cast<const TG *>(p.gate) + kept_gate + at.col[c]);
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            next.y[c] = tc_raw_load<T, VEC, LOOSE>(static_cast<const T *>(p.y) + row * p.ldy + at.col[c]);
            next.x[c] = tc_raw_load<float, VEC, LOOSE>(p.x + row * ldx + at.col[c]);
            next.dh[c] = tc_raw_load<T, VEC, LOOSE>(dh_rows + row * ld_dh + at.col[c]);
            next.d[c] = tc_raw_load<float, VEC, LOOSE>(d_rows + row * ld_d + at.col[c]);
        }
        next.st = *reinterpret_cast<const f32x4 *>(p.stats + row * 4);
    };
    float kg1[NC][VEC], kb1[NC][VEC], kg2[NC][VEC], kgt[NC][VEC];
    if (kKeep) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                kb1[c][j] = kg2[c][j] = 0.f;
                kgt[c][j] = 1.f;
            }
            tc_load_row<float, VEC, LOOSE>(p.g1 + at.col[c], kg1[c]);
            if (p.gate && p.b1) tc_load_row<float, VEC, LOOSE>(p.b1 + at.col[c], kb1[c]);
            if (p.g2) tc_load_row<float, VEC, LOOSE>(p.g2 + at.col[c], kg2[c]);
        }
    }
    if (kAhead && begin < end) {
        request(begin);
        arrived(kg1); arrived(kb1); arrived(kg2);
#pragma unroll
        for (int c = 0; c < NC; ++c) asm volatile("" : "+v"(next.y[c]), "+v"(next.x[c]), "+v"(next.dh[c]), "+v"(next.d[c]));
        asm volatile("" : "+v"(next.st));
    }
    for (long row = begin; row < end; ++row) {
        if (!kAhead) request(row);
        float yv[NC][VEC], xv[NC][VEC], dh[NC][VEC], d[NC][VEC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            tc_raw_widen<T, VEC>(next.y[c], yv[c]);
            tc_raw_widen<float, VEC>(next.x[c], xv[c]);
            tc_raw_widen<T, VEC>(next.dh[c], dh[c]);
            tc_raw_widen<float, VEC>(next.d[c], d[c]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[c][j] = p.dx_out ? d[c][j] : 0.f;
        }
        const f32x4 st = next.st;
        if (kKeep && fresh_gate) {
#pragma unroll
            for (int c = 0; c < NC; ++c) tc_raw_widen<TG, VEC>(next.gate[c], kgt[c]);
            arrived(kgt);
        }
        if (kAhead) request(min(row + 1, end - 1));
        // dx may be dx_out: every wave has its values of that before the barrier that is before the stores
        if (W > 1 && kAhead) {
            arrived(d);
            if (!p.g2) __syncthreads();
        }
        if (p.g2) {
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float g[VEC];
                if (!kKeep) tc_load_row<float, VEC, LOOSE>(p.g2 + at.col[c], g);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (kKeep) g[j] = kg2[c][j];
                    const float xh = (xv[c][j] - st[2]) * st[3];
                    acc[2][c][j] += dh[c][j] * xh;
                    acc[3][c][j] += dh[c][j];
                    const float q = dh[c][j] * g[j];
                    const float counted = at.counts(c, j) ? q : 0.f;
                    s1 += counted;
                    s2 += counted * xh;
                    xv[c][j] = xh;
                    dh[c][j] = q;
                }
            }
            team.sum2(s1, s2);
            const float m1 = p.rms ? 0.f : s1 * inv_e, m2 = s2 * inv_e;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[c][j] += st[3] * (dh[c][j] - m1 - xv[c][j] * m2);
        }
        if (!kAhead) {                       // a barrier of its own, where registers are too few to have the values early
            arrived(d);
            __syncthreads();
        }
        const long gate_row = gate_row_of(row);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float g[VEC], b[VEC], gt[VEC], o[VEC];
            if (!kKeep) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    b[j] = 0.f;
                    gt[j] = 1.f;
                }
                tc_load_row<float, VEC, LOOSE>(p.g1 + at.col[c], g);
                if (p.gate) tc_load_row<TG, VEC, LOOSE>(static_cast<const TG *>(p.gate) + gate_row + at.col[c], gt);
                if (p.gate && p.b1) tc_load_row<float, VEC, LOOSE>(p.b1 + at.col[c], b);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (kKeep) { g[j] = kg1[c][j]; b[j] = kb1[c][j]; gt[j] = kgt[c][j]; }
                const float yh = (yv[c][j] - st[0]) * st[1];
                dgt[c][j] += d[c][j] * (yh * g[j] + b[j]);
                const float dn = d[c][j] * gt[j];
                acc[0][c][j] += dn * yh;
                acc[1][c][j] += dn;
                const float q = dn * g[j];
                const float counted = at.counts(c, j) ? q : 0.f;
                s1 += counted;
                s2 += counted * yh;
                o[j] = p.res_scale * d[c][j];
                yv[c][j] = yh;
                d[c][j] = q;
            }
            tc_store_row<float, VEC, LOOSE>(p.dx + row * p.E + at.col[c], o);
        }
        team.sum2(s1, s2);
        const float m1 = p.rms ? 0.f : s1 * inv_e, m2 = s2 * inv_e;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = st[1] * (d[c][j] - m1 - yv[c][j] * m2);
            tc_store_row<T, VEC, LOOSE>(static_cast<T *>(p.dy) + row * p.E + at.col[c], o);
        }
        // the team's last row of a gate group: the group's gradient, or this team's part of it
        if (p.gate && p.teams_per_group == 0 && ((unsigned)row + 1) % (unsigned)p.rows_per_gate == 0) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float *to = p.d_gate + gate_row + at.col[c];
                if (at.skip[c] == 0) {
                    float old[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) old[j] = 0.f;
                    if (p.accumulate & 16) tc_load_row<float, VEC, LOOSE>(to, old);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) old[j] += dgt[c][j];
                    tc_store_row<float, VEC, LOOSE>(to, old);
                } else if (LOOSE) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (j >= at.skip[c]) to[j] = p.accumulate & 16 ? to[j] + dgt[c][j] : dgt[c][j];
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) dgt[c][j] = 0.f;
            }
        }
    }
    // workspace: [workgroups][4][E] vectors, then [teams][E] gate parts
    if (p.gate && p.teams_per_group > 0 && t < p.teams) {
        float *to = p.ws + (long)gridDim.x * 4 * p.E + (long)t * p.E;
#pragma unroll
        for (int c = 0; c < NC; ++c) tc_store_row<float, VEC, LOOSE>(to + at.col[c], dgt[c]);
    }
    float *to = p.ws + (long)blockIdx.x * 4 * p.E;
    if constexpr (W == 1) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (at.counts(c, j)) sums[wave * p.E + at.col[c] + j] = acc[v][c][j];
            __syncthreads();
            for (int i = threadIdx.x; i < p.E; i += 256) to[v * p.E + i] = (sums[i] + sums[p.E + i]) + (sums[2 * p.E + i] + sums[3 * p.E + i]);
            __syncthreads();
        }
    } else {
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int c = 0; c < NC; ++c) tc_store_row<float, VEC, LOOSE>(to + (long)v * p.E + at.col[c], acc[v][c]);
    }
}

// Column sums of the parts that the workgroups (v < 4: a vector's gradient) or the teams of a gate group (v - 4: the
// group) left: 64 columns per workgroup, 16 row lanes, added in a fixed order.
__global__ __launch_bounds__(1024) void gated_norm_join_kernel(const NormParams p, int workgroups, int groups) {
    __shared__ float red[16][64];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + c;
    for (int v = blockIdx.y; v < 4 + groups; v += gridDim.y) {
        const bool vec = v < 4;
        const int g = v - 4, n = vec ? workgroups : p.teams_per_group;
        float *out = vec ? p.d_vec[v] : p.d_gate + (long)g * p.E;
        const float *src = vec ? p.ws + (long)v * p.E : p.ws + (long)workgroups * 4 * p.E + (long)g * n * p.E;
        const long ld = vec ? 4L * p.E : p.E;
        if (!out) continue;
        float s = 0.f;
        if (col < p.E)
#pragma unroll 8
            for (int i = r; i < n; i += 16) s += src[i * ld + col];
        red[r][c] = s;
        __syncthreads();
        if (r == 0 && col < p.E) {
            for (int i = 1; i < 16; ++i) s += red[i][c];
            out[col] = (p.accumulate >> (vec ? v : 4)) & 1 ? out[col] + s : s;
        }
        __syncthreads();
    }
}

// How a row is laid over lanes: W waves a row, NC loads of VEC values a lane and operand.  Rows whose width or addresses do
// not allow aligned loads take the LOOSE form with unaligned ones.  The fewest waves of those built that hold the row in two
// loads, so that few lanes are left over (backward, 8192 bf16 rows of 2500: 5 waves 64 us, 8 82; of 5000: 10 158, 16 212).
// One wave a row needs no barrier, and four of them add their sums in LDS; more waves bring more of the chip to few rows.
// Forward, 768 wide, one / four waves: 131 rows f32 5.6 / 5.3 us, bf16 5.3 / 5.3, 65536 rows 140 / 154 and 114 / 137; 1024 wide
// 186 / 192 and 154 / 151: one wave up to there.
// Backward, one / three or four waves: 512 wide 131 rows 8.7 / 7.8, 1024 rows 12.3 / 11.6, 16384 rows f32 35.6 / 44.8; 768 wide 1024 rows
// 14.6 / 12.2, 8192 rows f32 30.1 / 28.3, bf16 25.5 / 26.5, 65536 rows 214 / 211 and 152 / 162; 600 wide 65536 rows 173 / 181 and 122 / 148.
struct Shape {
    int W, nc;
};
Shape row_shape(int E, bool one_wave) {
    int W = one_wave ? 1 : 4;
    if (!one_wave)
        for (const int more : {5, 6, 8, 10, 12, 16})
            if (E > 64 * VEC * 2 * W) W = more;
    return Shape{W, (E + 64 * VEC * W - 1) / (64 * VEC * W)};
}
Shape fwd_shape(int E) { return row_shape(E, E <= 1024); }
Shape bwd_shape(long M, int E) {
    const bool one_wave = E <= 512 || (E <= 768 && M >= 8192);
    return !one_wave && E <= 768 ? Shape{3, 1} : row_shape(E, one_wave);
}

struct BwdPlan {
    int teams, rows_per_team, teams_per_group, workgroups;
    size_t bytes;
};
BwdPlan bwd_plan(int M, int E, int G) {
    BwdPlan w{};
    const int W = bwd_shape(M, E).W;
    const int per_wg = W == 1 ? 4 : 1;
    // Teams: as many workgroups as the CUs take alike, one each, or two of three or four waves (16384 x 768 bf16: 512 teams 38.5 us,
    // 683 40.1, 1024 37.5, 1365 44.1; 16384 x 4096: 256 189, 512 202, 683 213).  Every workgroup leaves 4 E sums to be written and
    // joined, so it takes a few rows even where the chip is not full (1024 x 768: 1 row 17.7 us, 2 12.9, 4 11.8, 8 13.9).
    const int want = W == 1 ? 1024 : W <= 4 ? 512 : 256;
    const int least = M >= 768 ? 4 : M >= 192 ? 2 : 1;
    int rows = (int)(((long)M + want - 1) / want);
    rows = rows > least ? rows : least;
    const int group = G > 0 ? M / G : 0;
    if (G == 0 || group <= rows) {
        w.rows_per_team = G == 0 ? rows : rows / group * group;
        w.teams = (int)(((long)M + w.rows_per_team - 1) / w.rows_per_team);
    } else {
        w.teams_per_group = (int)(((long)group + rows - 1) / rows);
        w.rows_per_team = (int)(((long)group + w.teams_per_group - 1) / w.teams_per_group);
        w.teams = G * w.teams_per_group;
    }
    w.workgroups = (w.teams + per_wg - 1) / per_wg;
    w.bytes = ((size_t)w.workgroups * 4 + (w.teams_per_group > 0 ? w.teams : 0)) * E * sizeof(float);
    return w;
}

int check_common(const char *who, int dtype, int gate_dtype, const void *gate, long M, int E, int G) {
    TC_REQUIRE(dtype == TC_F32 || dtype == TC_BF16, "%s: bad dtype %d", who, dtype);
    TC_REQUIRE(M > 0 && M <= 0x7fffffffL && E > 0 && E <= 8192, "%s: bad shape M=%ld E=%d (E <= 8192)", who, M, E);
    TC_REQUIRE((gate != nullptr) == (G > 0), "%s: a gate and its %d rows go together", who, G);
    TC_REQUIRE(G >= 0 && (G == 0 || M % G == 0), "%s: %d gate rows do not divide %ld rows", who, G, M);
    TC_REQUIRE(gate_dtype == TC_F32 || (gate_dtype == TC_BF16 && dtype == TC_BF16), "%s: bad gate type %d", who, gate_dtype);
    TC_REQUIRE((uintptr_t)gate % (gate_dtype == TC_BF16 ? 2 : 4) == 0, "%s: misaligned gate", who);
    return TC_OK;
}

}  // namespace

// the shapes that fwd_shape and bwd_shape name, as W * 10 + NC
#define TC_GN_COMMON(T, TG, LOOSE)                                                              \
            case 11: TC_GN(T, TG, LOOSE, 1, 1); break;                                          \
            case 12: TC_GN(T, TG, LOOSE, 1, 2); break;                                          \
            case 13: TC_GN(T, TG, LOOSE, 1, 3); break;                                          \
            case 42: TC_GN(T, TG, LOOSE, 4, 2); break;                                          \
            case 52: TC_GN(T, TG, LOOSE, 5, 2); break;                                          \
            case 62: TC_GN(T, TG, LOOSE, 6, 2); break;                                          \
            case 82: TC_GN(T, TG, LOOSE, 8, 2); break;                                          \
            case 102: TC_GN(T, TG, LOOSE, 10, 2); break;                                        \
            case 122: TC_GN(T, TG, LOOSE, 12, 2); break;                                        \
            default: TC_GN(T, TG, LOOSE, 16, 2); break;
#define TC_GN_FWD(T, TG, LOOSE)                                                                 \
    do {                                                                                        \
        if (E < VEC) TC_GN_V(T, TG, false, 1, 1, 1);                                            \
        else switch (sh.W * 10 + sh.nc) {                                                       \
            case 14: TC_GN(T, TG, LOOSE, 1, 4); break;                                          \
            TC_GN_COMMON(T, TG, LOOSE)                                                          \
        }                                                                                       \
    } while (0)
#define TC_GN_BWD(T, TG, LOOSE)                                                                 \
    do {                                                                                        \
        if (E < VEC) TC_GN_V(T, TG, false, 1, 1, 1);                                            \
        else switch (sh.W * 10 + sh.nc) {                                                       \
            case 31: TC_GN(T, TG, LOOSE, 3, 1); break;                                          \
            case 41: TC_GN(T, TG, LOOSE, 4, 1); break;                                          \
            TC_GN_COMMON(T, TG, LOOSE)                                                          \
        }                                                                                       \
    } while (0)
#define TC_GN_L(K, T, TG)                                                                       \
    do {                                                                                        \
        if (loose) K(T, TG, true);                                                              \
        else K(T, TG, false);                                                                   \
    } while (0)
#define TC_GN_T(K)                                                                              \
    do {                                                                                        \
        if (dtype == TC_F32) TC_GN_L(K, float, float);                                          \
        else if (gate_dtype == TC_F32) TC_GN_L(K, uint16_t, float);                             \
        else TC_GN_L(K, uint16_t, uint16_t);                                                    \
    } while (0)

extern "C" int tc_gated_residual_norm_fwd(int dtype, const void *y, long ldy, const float *x, long ldx, const float *post_gamma,
                                          const float *post_beta, int gate_dtype, const void *gate, int G, float res_scale,
                                          const float *pre_gamma, const float *pre_beta, float *x_out, void *h, float *stats,
                                          long M, int E, int rms, float post_eps, float pre_eps, void *stream) {
    const int rc = check_common("tc_gated_residual_norm_fwd", dtype, gate_dtype, gate, M, E, G);
    if (rc != TC_OK) return rc;
    TC_REQUIRE(y && x && post_gamma && x_out, "tc_gated_residual_norm_fwd: null operand");
    TC_REQUIRE((pre_gamma != nullptr) == (h != nullptr) && (pre_gamma || !pre_beta),
               "tc_gated_residual_norm_fwd: the second norm's vectors and h go together");
    TC_REQUIRE(ldy >= E && ldx >= E, "tc_gated_residual_norm_fwd: row stride below E");
    const int esz = dtype == TC_BF16 ? 2 : 4;
    TC_REQUIRE((uintptr_t)y % esz == 0 && (uintptr_t)h % esz == 0 && tc_aligned16(stats) &&
                   ((uintptr_t)x | (uintptr_t)x_out | (uintptr_t)post_gamma | (uintptr_t)post_beta | (uintptr_t)pre_gamma |
                    (uintptr_t)pre_beta) % 4 == 0,
               "tc_gated_residual_norm_fwd: misaligned operand (stats: 16 bytes)");
    NormParams p{};
    p.y = y; p.x = x; p.gate = gate;
    p.g1 = post_gamma; p.b1 = post_beta; p.g2 = pre_gamma; p.b2 = pre_beta;
    p.x_out = x_out; p.h = h; p.stats = stats;
    p.ldy = ldy; p.ldx = ldx;
    p.M = (int)M; p.E = E; p.rms = rms;
    p.rows_per_gate = G > 0 ? (int)(M / G) : (int)M;
    p.res_scale = res_scale; p.eps1 = post_eps; p.eps2 = pre_eps;
    const int g_esz = gate_dtype == TC_BF16 ? 2 : 4;
    const bool loose = !(tc_rows_aligned(y, ldy, esz, VEC) && tc_rows_aligned(x, ldx, 4, VEC) && tc_rows_aligned(gate, E, g_esz, VEC) &&
               tc_rows_aligned(h, E, esz, VEC) && tc_rows_aligned(x_out, E, 4, VEC) && tc_rows_aligned(post_gamma, 0, 4, VEC) &&
               tc_rows_aligned(post_beta, 0, 4, VEC) && tc_rows_aligned(pre_gamma, 0, 4, VEC) && tc_rows_aligned(pre_beta, 0, 4, VEC));
    const Shape sh = fwd_shape(E);
    const int per_wg = sh.W == 1 ? 4 : 1;
    long blocks = (M + per_wg - 1) / per_wg;
    // rows are walked with the grid's stride: a launch holds fewer than 2^32 threads, and teams that ask ahead fill the chip once
    const long most = sh.W > 8 ? 256 : sh.W > 4 ? 512 : 1L << 21;
    if (blocks > most) blocks = most;
    hipStream_t s = static_cast<hipStream_t>(stream);
    TcProfScope prof(TC_PROF_LAYERNORM, s, (double)M * E * (2 * esz + 8));
#define TC_GN_V(T, TG, L, WW, N, V) \
    TC_LAUNCH((gated_norm_kernel<T, TG, L, WW, N, V>), dim3((unsigned)blocks), dim3(WW == 1 ? 256 : 64 * WW), 0, s, p)
#define TC_GN(T, TG, L, WW, N) TC_GN_V(T, TG, L, WW, N, VEC)
    TC_GN_T(TC_GN_FWD);
#undef TC_GN
#undef TC_GN_V
    TC_CHECK_LAUNCH("tc_gated_residual_norm_fwd");
    return TC_OK;
}

extern "C" size_t tc_gated_residual_norm_bwd_workspace_bytes(long M, int E, int G) {
    if (M <= 0 || M > 0x7fffffffL || E <= 0 || E > 8192 || G < 0 || (G > 0 && M % G != 0)) return 0;
    return bwd_plan((int)M, E, G).bytes;
}

extern "C" int tc_gated_residual_norm_bwd(int dtype, const void *dh, long ld_dh, const float *dx_out, long ld_dxo, const void *y,
                                          long ldy, const float *x_out, long ldx, const float *stats, const float *post_gamma,
                                          const float *post_beta, int gate_dtype, const void *gate, int G, float res_scale,
                                          const float *pre_gamma, void *dy, float *dx, float *d_post_gamma,
                                          float *d_post_beta, float *d_gate, float *d_pre_gamma, float *d_pre_beta,
                                          int accumulate, long M, int E, int rms, void *workspace, size_t workspace_bytes,
                                          void *stream) {
    const int rc = check_common("tc_gated_residual_norm_bwd", dtype, gate_dtype, gate, M, E, G);
    if (rc != TC_OK) return rc;
    TC_REQUIRE(y && x_out && stats && post_gamma && dy && dx && workspace, "tc_gated_residual_norm_bwd: null operand");
    TC_REQUIRE((pre_gamma != nullptr) == (dh != nullptr) && (pre_gamma || (!d_pre_gamma && !d_pre_beta)),
               "tc_gated_residual_norm_bwd: the second norm's vector, its gradients and dh go together");
    TC_REQUIRE(dh || dx_out, "tc_gated_residual_norm_bwd: neither dh nor dx_out");
    TC_REQUIRE((gate != nullptr) == (d_gate != nullptr), "tc_gated_residual_norm_bwd: a gate and its gradient go together");
    TC_REQUIRE(ldy >= E && ldx >= E && (!dh || ld_dh >= E) && (!dx_out || ld_dxo >= E),
               "tc_gated_residual_norm_bwd: row stride below E");
    const int esz = dtype == TC_BF16 ? 2 : 4;
    TC_REQUIRE(((uintptr_t)y | (uintptr_t)dh | (uintptr_t)dy) % esz == 0 && tc_aligned16(stats) && tc_aligned16(workspace) &&
                   ((uintptr_t)x_out | (uintptr_t)dx_out | (uintptr_t)dx | (uintptr_t)post_gamma | (uintptr_t)post_beta |
                    (uintptr_t)pre_gamma | (uintptr_t)d_post_gamma | (uintptr_t)d_post_beta | (uintptr_t)d_gate |
                    (uintptr_t)d_pre_gamma | (uintptr_t)d_pre_beta) % 4 == 0,
               "tc_gated_residual_norm_bwd: misaligned operand (stats and workspace: 16 bytes)");
    const size_t need = tc_gated_residual_norm_bwd_workspace_bytes(M, E, G);
    if (workspace_bytes < need) {
        tc_set_error("tc_gated_residual_norm_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return TC_ENOSPC;
    }
    // the sums are added by workgroups of their own: one buffer for two of them would lose one
    const float *const sums[5] = {d_post_gamma, d_post_beta, d_pre_gamma, d_pre_beta, d_gate};
    for (int a = 0; a < 5; ++a)
        for (int b = 0; b < a; ++b) {
            const uintptr_t from_a = (uintptr_t)sums[a], from_b = (uintptr_t)sums[b];
            const uintptr_t len_a = (uintptr_t)E * 4 * (a == 4 ? G : 1), len_b = (uintptr_t)E * 4;
            TC_REQUIRE(!sums[a] || !sums[b] || from_a + len_a <= from_b || from_b + len_b <= from_a,
                       "tc_gated_residual_norm_bwd: gradients of the vectors overlap");
        }
    const int g_esz = gate_dtype == TC_BF16 ? 2 : 4;
    const bool loose = !(tc_rows_aligned(y, ldy, esz, VEC) && tc_rows_aligned(x_out, ldx, 4, VEC) && tc_rows_aligned(gate, E, g_esz, VEC) &&
               (!dh || tc_rows_aligned(dh, ld_dh, esz, VEC)) && (!dx_out || tc_rows_aligned(dx_out, ld_dxo, 4, VEC)) &&
               tc_rows_aligned(dy, E, esz, VEC) && tc_rows_aligned(dx, E, 4, VEC) && tc_rows_aligned(d_gate, E, 4, VEC) &&
               tc_rows_aligned(post_gamma, 0, 4, VEC) && tc_rows_aligned(post_beta, 0, 4, VEC) && tc_rows_aligned(pre_gamma, 0, 4, VEC));
    const Shape sh = bwd_shape(M, E);
    const BwdPlan w = bwd_plan((int)M, E, G);
    NormParams p{};
    p.y = y; p.x = x_out; p.gate = gate; p.dh = dh; p.dx_out = dx_out;
    p.stats = const_cast<float *>(stats);
    p.g1 = post_gamma; p.b1 = post_beta; p.g2 = pre_gamma;
    p.dy = dy; p.dx = dx; p.d_gate = d_gate;
    p.ws = static_cast<float *>(workspace);
    p.d_vec[0] = d_post_gamma; p.d_vec[1] = d_post_beta; p.d_vec[2] = d_pre_gamma; p.d_vec[3] = d_pre_beta;
    p.accumulate = accumulate;
    p.ldy = ldy; p.ldx = ldx; p.ld_dh = ld_dh; p.ld_dxo = ld_dxo;
    p.M = (int)M; p.E = E; p.rms = rms;
    p.rows_per_gate = G > 0 ? (int)(M / G) : (int)M;
    p.res_scale = res_scale;
    p.teams = w.teams; p.rows_per_team = w.rows_per_team; p.teams_per_group = w.teams_per_group;
    hipStream_t s = static_cast<hipStream_t>(stream);
    TcProfScope prof(TC_PROF_LAYERNORM, s, (double)M * E * (3 * esz + 12));
#define TC_GN_V(T, TG, L, WW, N, V)                                                                                        \
    TC_LAUNCH((gated_norm_bwd_kernel<T, TG, L, WW, N, V>), dim3((unsigned)w.workgroups), dim3(WW == 1 ? 256 : 64 * WW),     \
              WW == 1 ? 16 * (size_t)E : 0, s, p)
#define TC_GN(T, TG, L, WW, N) TC_GN_V(T, TG, L, WW, N, VEC)
    TC_GN_T(TC_GN_BWD);
#undef TC_GN
#undef TC_GN_V
    const int groups = w.teams_per_group > 0 ? G : 0;
    const int tall = 4 + groups < 1024 ? 4 + groups : 1024;
    TC_LAUNCH(gated_norm_join_kernel, dim3((E + 63) / 64, tall), dim3(1024), 0, s, p, w.workgroups, groups);
    TC_CHECK_LAUNCH("tc_gated_residual_norm_bwd");
    return TC_OK;
}
